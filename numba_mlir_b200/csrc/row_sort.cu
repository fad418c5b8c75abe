// Entries sorted by group: the stable order of the row operators (rows.cu).
//
// A least-significant-digit radix sort of (key, entry) pairs, key = id for an
// id inside [0, groups) and `groups` for every other one, over
// bits(groups) bits in the fewest passes of at most 10 bits each: one pass up
// to 1023 groups (experts), two up to a million (a vocabulary).  Nothing
// depends on the order in which blocks or atomics run: a block counts its own
// entries, counts are added up in block order, and the rank of an entry among
// the equal digits of its warp's 32 comes from votes over the warp.
//
// What it costs is latency, not bandwidth (an entry is 8 bytes), so the number
// of dependent steps is what the three forms differ in.  Up to 2048 entries (4096
// of many groups) are not sorted in passes at all: every position is counted.  Up to about a
// million take a launch that counts tiles of 1024 to 8192 entries and one a pass
// that scatters them: each block adds up the counts of all blocks for itself (at
// most 148 of them), and counts its entries for the pass after it at the places
// they go to.  Beyond that a launch a pass adds the counts up.
#include "rows_host.h"

#include <atomic>
#include <type_traits>

#define GPUX_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

constexpr int kMaxDigitBits = 10;
constexpr int kBins = 1 << kMaxDigitBits;
constexpr unsigned kAll = 0xffffffffu;

struct Ids {
  const void *data;
  int bytes;
  uint32_t groups;
  __device__ __forceinline__ int64_t raw(int64_t i) const {
    return bytes == 8 ? __ldg(static_cast<const long long *>(data) + i)
                      : (int64_t)__ldg(static_cast<const int *>(data) + i);
  }
  __device__ __forceinline__ uint32_t cooked(int64_t id) const {
    return id >= 0 && id < (int64_t)groups ? (uint32_t)id : groups;
  }
  __device__ __forceinline__ uint32_t key(int64_t i) const { return cooked(raw(i)); }
};

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

constexpr int kThreads = 1024;
constexpr int kThreadBits = 10, kWarpBits = 5, kWarps = kThreads / 32;
constexpr int kMostPerThread = 8;
constexpr int kMostBlocks = 148;

struct Results {
  int32_t *order;
  uint32_t *keys;
  int32_t *place;
  int32_t *offsets;
};

// Words that a kernel's sorting blocks set to zero on the way.
struct Clear {
  uint32_t *words;
  int64_t count;
  __device__ __forceinline__ void run(int blocks) const {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (int64_t)blocks * blockDim.x)
      words[i] = 0;
  }
};

// Rows that a kernel sets to zero in blocks of their own, behind `first`: up to
// 64 KB a block.
constexpr int kFillBytes = 65536;
struct Fill {
  unsigned char *data; // the first of the rows
  int64_t accesses;    // in all
  int64_t per_row, stride;
  int unit;
  int first;
  int head, tail;      // bytes before and behind, where rows follow one another
  __device__ __forceinline__ bool run() const {
    if ((int)blockIdx.x < first)
      return false;
    const int64_t per_block = kFillBytes / unit;
    if ((int)blockIdx.x == first && (int)threadIdx.x * 2 < head + tail) {
      const int at = (int)threadIdx.x * 2;
      *reinterpret_cast<short *>(at < head ? data - head + at : data + accesses * unit + (at - head)) = 0;
    }
    const int64_t begin = (int64_t)(blockIdx.x - first) * per_block, end = min(begin + per_block, accesses);
    for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
      // rows that follow one another are one long row
      const int64_t row = per_row == accesses ? 0 : i / per_row;
      unsigned char *to = data + row * stride + (i - row * per_row) * unit;
      if (unit == 16)
        *reinterpret_cast<int4 *>(to) = make_int4(0, 0, 0, 0);
      else if (unit == 8)
        *reinterpret_cast<int2 *>(to) = make_int2(0, 0);
      else if (unit == 4)
        *reinterpret_cast<int *>(to) = 0;
      else
        *reinterpret_cast<short *>(to) = 0;
    }
    return true;
  }
};

// Where a block's entries go among its entries of each digit.  An entry's rank
// is made of three: among the equal digits of its warp (rank), in the warps of
// its part before that (counts), in the parts before that (parts).  A part is a
// share of the warps that one thread adds up, for two digits at a time: a block's
// counts fit 16 bits, and two of them add in one word.
struct Digits {
  uint16_t *counts;  // [warps][bins]
  uint16_t *parts;   // [parts][bins]
  int bins, bin_bits, shift, part_bits; // 1 << part_bits warps to a part
  __device__ __forceinline__ uint32_t of(uint32_t key) const { return (key >> shift) & (uint32_t)(bins - 1); }

  __device__ __forceinline__ Digits(uint16_t *counts, uint16_t *parts, int bin_bits, int shift)
      : counts(counts), parts(parts), bins(1 << bin_bits), bin_bits(bin_bits), shift(shift),
        // kThreads / (bins / 2) parts, but not more than warps
        part_bits(max(kWarpBits - (kThreadBits - bin_bits + 1), 0)) {}

  __device__ __forceinline__ void clear() const {
    uint32_t *words = reinterpret_cast<uint32_t *>(counts);
    for (int i = threadIdx.x; i < kWarps * bins / 2; i += kThreads)
      words[i] = 0;
  }

  // Rank of this lane's digit among the equal digits of the lanes before it and
  // of the calls before this one.  The lanes with the same digit find one
  // another bit by bit; the first of them moves the warp's count.
  __device__ __forceinline__ uint32_t rank(uint32_t digit, bool live) const {
    const int lane = threadIdx.x & 31;
    unsigned peers = __ballot_sync(kAll, live);
    for (int b = 1; b < bins; b <<= 1) {
      const unsigned ones = __ballot_sync(kAll, digit & b);
      peers &= digit & b ? ones : ~ones;
    }
    uint16_t *mine = counts + (threadIdx.x >> 5) * bins + digit;
    const uint32_t before = live ? *mine : 0;
    __syncwarp();
    const unsigned lower = peers & ((1u << lane) - 1);
    if (live && lower == 0)
      *mine = (uint16_t)(before + __popc(peers));
    __syncwarp();
    return before + __popc(lower);
  }

  // Adds the warps' counts up, four at a time, then the parts', for `before`.
  // Between two barriers of the caller's.
  __device__ __forceinline__ void add_up() const {
    uint32_t *pairs = reinterpret_cast<uint32_t *>(counts), *sums = reinterpret_cast<uint32_t *>(parts);
    const int half = bins / 2, count = kWarps >> part_bits, rows = 1 << part_bits;
    const int pair = threadIdx.x & (half - 1), part = threadIdx.x >> (bin_bits - 1);
    if (part < count) {
      uint32_t sum = 0;
      for (int w = part * rows; w < (part + 1) * rows; w += 4) {
        uint32_t c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          c[u] = u < rows ? pairs[(w + u) * half + pair] : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (u < rows)
            pairs[(w + u) * half + pair] = sum;
          sum += c[u];
        }
      }
      sums[part * half + pair] = sum;
    }
    __syncthreads();
    if (part == 0) {
      uint32_t sum = 0;
      for (int q = 0; q < count; q += 4) {
        uint32_t c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          c[u] = q + u < count ? sums[(q + u) * half + pair] : 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (q + u < count)
            sums[(q + u) * half + pair] = sum;
          sum += c[u];
        }
      }
    }
  }
  __device__ __forceinline__ uint32_t before(uint32_t digit) const {
    const int warp = threadIdx.x >> 5;
    return parts[(warp >> part_bits << bin_bits) + digit] + counts[(warp << bin_bits) + digit];
  }
};

// ---- few entries ------------------------------------------------------------------
// No passes: a warp finds an entry's position by counting the entries of smaller
// keys and the earlier ones of the same key.  That is a comparison for every pair
// of entries, but they depend on nothing and fill the machine; a radix sort of
// the same entries in one block took 4 to 8 us a pass.
constexpr int kFew = 4096, kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewGroups = 1023; // more groups: their offsets come from a launch of their own

__global__ void __launch_bounds__(kFewThreads)
    nmb_sort_few(const Ids ids, int n, int blocks, const Results res, const Clear clear, const Fill fill) {
  nmb::rows::let_next_begin();
  if (fill.run())
    return;
  __shared__ __align__(16) uint32_t keys[kFew];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int padded = (n + 127) / 128 * 128; // whole rows of four keys a lane, the rest above every key
  for (int i = threadIdx.x; i < padded; i += kFewThreads)
    keys[i] = i < n ? ids.key(i) : 0xffffffffu;
  clear.run(blocks);
  __syncthreads();
  const int e = (int)blockIdx.x * kFewWarps + warp;
  if (e < n) {
    const uint32_t key = keys[e];
    int before = 0;
    for (int i = lane * 4; i < padded; i += 128) {
      const uint4 k = *reinterpret_cast<const uint4 *>(keys + i);
      // keys of earlier entries count when equal, too
      before += (k.x < key + (i < e)) + (k.y < key + (i + 1 < e)) + (k.z < key + (i + 2 < e)) +
                (k.w < key + (i + 3 < e));
    }
    before = __reduce_add_sync(kAll, before);
    if (lane == 0) {
      if (res.order)
        res.order[before] = e;
      if (res.keys)
        res.keys[before] = key;
      if (res.place)
        res.place[e] = before;
    }
  }
  if (res.offsets)
    for (int g = (int)blockIdx.x * kFewWarps + warp; g <= (int)ids.groups; g += blocks * kFewWarps) {
      int before = 0;
      for (int i = lane * 4; i < padded; i += 128) {
        const uint4 k = *reinterpret_cast<const uint4 *>(keys + i);
        before += (k.x < (uint32_t)g) + (k.y < (uint32_t)g) + (k.z < (uint32_t)g) + (k.w < (uint32_t)g);
      }
      before = __reduce_add_sync(kAll, before);
      if (lane == 0)
        res.offsets[g] = before;
    }
}

// ---- many blocks ----------------------------------------------------------------
// A block's counts are 16-bit (it has 8192 entries at most), two digits to a
// word.  With `added` they hold the entries of the blocks before it, in words.
struct Pass {
  Ids ids;                 // the first pass reads its keys here (keysIn == nullptr)
  const uint32_t *keysIn;
  const int32_t *entriesIn;
  uint32_t *counts;        // [blocks][bins / 2], of this pass
  uint32_t *next;          // the same of the pass after it, zero, or null
  uint32_t *added;         // [blocks][bins] and then [bins] totals, or null
  int64_t n;
  int blocks, shift, bins, digit_bits;
  // an entry's key in two steps: what is read, and what is made of it
  __device__ __forceinline__ int64_t raw(int64_t i) const { return keysIn ? (int64_t)nmb::rows::made(keysIn + i) : ids.raw(i); }
  __device__ __forceinline__ uint32_t cooked(int64_t id) const { return ids.cooked(id); }
  __device__ __forceinline__ uint32_t key(int64_t i) const { return cooked(raw(i)); }
  __device__ __forceinline__ uint32_t digit(uint32_t k) const { return (k >> shift) & (uint32_t)(bins - 1); }
};

// Counts of the first pass; those of a later one are made by the scatter before
// it.  Also clears them, and the caller's words.
template <int PER>
__global__ void __launch_bounds__(kThreads) nmb_sort_count(const Pass p, const Clear next, const Clear clear,
                                                            const Fill fill) {
  nmb::rows::let_next_begin();
  if (fill.run())
    return;
  __shared__ uint32_t count[kBins / 2];
  const int64_t base = (int64_t)blockIdx.x * kThreads * PER + threadIdx.x;
  uint32_t key[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u)
    key[u] = base + u * kThreads < p.n ? p.key(base + u * kThreads) : 0;
  next.run(p.blocks);
  clear.run(p.blocks);
  for (int b = threadIdx.x; b < p.bins / 2; b += kThreads)
    count[b] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (base + u * kThreads < p.n) {
      const uint32_t d = p.digit(key[u]);
      atomicAdd(&count[d >> 1], d & 1 ? 0x10000u : 1u);
    }
  __syncthreads();
  for (int b = threadIdx.x; b < p.bins / 2; b += kThreads)
    p.counts[(int64_t)blockIdx.x * (p.bins / 2) + b] = count[b];
}

// A warp per digit: added[b][d] <- sum of counts[0..b)[d], and the totals.
constexpr int kAddThreads = 256;
__global__ void __launch_bounds__(kAddThreads) nmb_sort_add(const Pass p) {
  const int lane = threadIdx.x & 31, d = blockIdx.x * (kAddThreads / 32) + (threadIdx.x >> 5);
  if (d >= p.bins)
    return;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < p.blocks; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t pair = b < p.blocks ? p.counts[(int64_t)b * (p.bins / 2) + (d >> 1)] : 0;
    const uint32_t v = d & 1 ? pair >> 16 : pair & 0xffff;
    uint32_t inc = v;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t t = __shfl_up_sync(kAll, inc, s);
      if (lane >= s)
        inc += t;
    }
    if (b < p.blocks)
      p.added[(int64_t)b * p.bins + d] = carry + inc - v;
    carry += __shfl_sync(kAll, inc, 31);
  }
  if (lane == 0)
    p.added[(int64_t)p.blocks * p.bins + d] = carry;
}

template <int PER>
__global__ void __launch_bounds__(kThreads)
    nmb_sort_scatter(const Pass p, uint32_t *keysOut, int32_t *entriesOut, int32_t *place, int32_t *offsets,
                     const Fill fill) {
  nmb::rows::let_next_begin();
  if (fill.run())
    return;
  extern __shared__ uint32_t smem[];
  uint32_t *start = smem;                   // [bins]
  uint32_t *sums = start + kBins;           // [32]
  uint2 *shares = reinterpret_cast<uint2 *>(sums + 32); // [2][threads]: a thread's blocks before this one, all its blocks
  uint16_t *counts = reinterpret_cast<uint16_t *>(shares + 2 * kThreads);
  uint16_t *parts = counts + kWarps * kBins; // [parts][bins]: 2 * kThreads at most
  const Digits dg(counts, parts, p.digit_bits, p.shift);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t begin = ((int64_t)blockIdx.x * kWarps + warp) * PER * 32 + lane;
  uint32_t key[PER], rank[PER];
  int32_t entry[PER];
  dg.clear();
  nmb::rows::wait_for_previous();
  // counts of all blocks: a thread adds up every share-th block for two digits,
  // sixteen loads in flight (one by one they took 15 of the kernel's 19 us at
  // 131072 entries: an L2 access costs about 700 cycles), and the entries' own
  // with the first of them
  const int pairs = p.bins / 2, share = kThreads >> (p.digit_bits - 1), part = tid >> (p.digit_bits - 1);
  const uint32_t *from = p.counts + (tid & (pairs - 1));
  uint32_t c[16];
  auto read_counts = [&](int b0) {
#pragma unroll
    for (int u = 0; u < 16; ++u)
      c[u] = b0 + u * share < p.blocks ? nmb::rows::made(from + (int64_t)(b0 + u * share) * pairs) : 0;
  };
  if (!p.added)
    read_counts(part);
  int64_t id[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int64_t i = begin + u * 32;
    id[u] = i < p.n ? p.raw(i) : 0;
    entry[u] = i < p.n && p.entriesIn ? nmb::rows::made(p.entriesIn + i) : (int32_t)i;
  }
  if (!p.added) {
    uint2 mine = make_uint2(0, 0), all = make_uint2(0, 0);
    for (int b0 = part;;) {
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const uint32_t lo = c[u] & 0xffff, hi = c[u] >> 16;
        all.x += lo;
        all.y += hi;
        mine.x += b0 + u * share < (int)blockIdx.x ? lo : 0;
        mine.y += b0 + u * share < (int)blockIdx.x ? hi : 0;
      }
      b0 += 16 * share;
      if (b0 >= p.blocks)
        break;
      read_counts(b0);
    }
    shares[tid] = mine;
    shares[kThreads + tid] = all;
  }
#pragma unroll
  for (int u = 0; u < PER; ++u)
    key[u] = p.cooked(id[u]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u)
    rank[u] = dg.rank(dg.of(key[u]), begin + u * 32 < p.n);
  // where digit tid's entries begin: behind all smaller digits, and behind the
  // digit's entries in the blocks before this one
  uint32_t blocks_before = 0, total = 0;
  if (tid < p.bins) {
    if (p.added) {
      blocks_before = p.added[(int64_t)blockIdx.x * p.bins + tid];
      total = p.added[(int64_t)p.blocks * p.bins + tid];
    } else {
      const uint32_t *words = reinterpret_cast<const uint32_t *>(shares);
#pragma unroll 4
      for (int s = 0; s < share; ++s) {
        blocks_before += words[s * p.bins + tid];
        total += words[2 * kThreads + s * p.bins + tid];
      }
    }
  }
  const uint32_t digit_start = block_prefix(total, sums); // also: every warp's counts are done
  if (offsets && blockIdx.x == 0 && tid <= (int)p.ids.groups && tid < p.bins)
    offsets[tid] = (int32_t)digit_start;
  dg.add_up();
  if (tid < p.bins)
    start[tid] = digit_start + blocks_before;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (begin + u * 32 < p.n) {
      const uint32_t d = dg.of(key[u]), at = start[d] + dg.before(d) + rank[u];
      if (keysOut)
        keysOut[at] = key[u];
      if (entriesOut)
        entriesOut[at] = entry[u];
      if (place)
        place[entry[u]] = (int32_t)at;
      if (p.next) { // the digit that the entry has in the next pass, in the block that will read it there
        const uint32_t e = (key[u] >> (p.shift + p.digit_bits)) & (uint32_t)(p.bins - 1);
        atomicAdd(p.next + (int64_t)(at / (kThreads * PER)) * pairs + (e >> 1), e & 1 ? 0x10000u : 1u);
      }
    }
  }
}
constexpr int kScatterBytes = (kBins + 32) * 4 + 2 * kThreads * 8 + kWarps * kBins * 2 + 2 * kThreads * 2;

// offsets[g] = position of the first key >= g, for the sorts of several passes.
constexpr int kOffsetThreads = 256;
__global__ void __launch_bounds__(kOffsetThreads)
    nmb_sort_offsets(const uint32_t *keys, int64_t n, int64_t groups, int32_t *offsets) {
  const int64_t g = (int64_t)blockIdx.x * kOffsetThreads + threadIdx.x;
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

__global__ void __launch_bounds__(kOffsetThreads) nmb_sort_nothing(int64_t groups, int32_t *offsets) {
  const int64_t g = (int64_t)blockIdx.x * kOffsetThreads + threadIdx.x;
  if (g <= groups)
    offsets[g] = 0;
}

int bitsOf(int64_t groups) {
  int b = 1;
  while ((int64_t(1) << b) <= groups)
    ++b;
  return b; // keys are 0 .. groups
}

int passesOf(int64_t groups) { return (bitsOf(groups) + kMaxDigitBits - 1) / kMaxDigitBits; }

size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Counting beats one pass of a sort up to 2048 entries (4.8 against 6.5 us, at
// 4096 10.1 against 7), two passes up to 4096 (13.7 against 16).
bool isFew(int64_t n, int64_t groups) { return n <= (groups > kFewGroups ? kFew : kFew / 2); }

// Entries per thread of the many blocks: the fewest that keep them at 148 at
// most, and never more than 8.
int perThread(int64_t n) {
  int per = 1;
  while (per < kMostPerThread && n > (int64_t)per * kThreads * kMostBlocks)
    per *= 2;
  return per;
}
int64_t manyBlocks(int64_t n) {
  const int64_t tile = (int64_t)perThread(n) * kThreads;
  return (n + tile - 1) / tile;
}

// Counts of the digits of all blocks, of one pass.
size_t countBytes(size_t blocks) { return padded(blocks * kBins * 2); }

// The rows that a launch of `first` sorting blocks clears: 48 MB at most, about
// what the other multiprocessors write meanwhile (the gradient of 32768 rows into
// 131072 of 4096 bfloat16: 239 us without, 225 us at 32 and at 48 MB, 234 us at
// 96 MB; 777 rows into 10007 of 1000 float32: 17.5, 14.4, 13.3, 13.2 us).
constexpr int64_t kFillMost = 48 << 20;
Fill takeRows(nmb::rows::Clearing *c, int first, unsigned *blocks) {
  *blocks = (unsigned)first;
  if (!c || c->left == 0 || c->rowBytes == 0)
    return Fill{nullptr, 0, 1, 0, 16, first, 0, 0};
  int64_t rows = kFillMost / c->rowBytes;
  rows = rows < 1 ? 1 : rows < c->left ? rows : c->left;
  c->left -= rows;
  unsigned char *data = c->data + c->left * c->stride;
  Fill fill{data, rows * (c->rowBytes / c->unit), c->rowBytes / c->unit, c->stride, c->unit, first, 0, 0};
  if (c->stride == c->rowBytes) {
    // one long row: 16-byte stores whatever the rows' own boundaries
    const int64_t bytes = rows * c->rowBytes;
    const int64_t head = (int64_t)(-reinterpret_cast<intptr_t>(data) & 15);
    fill.head = (int)(head < bytes ? head : bytes);
    fill.data = data + fill.head;
    fill.unit = 16;
    fill.accesses = fill.per_row = (bytes - fill.head) / 16;
    fill.tail = (int)((bytes - fill.head) % 16);
  }
  const int64_t perBlock = kFillBytes / fill.unit, fillBlocks = (fill.accesses + perBlock - 1) / perBlock;
  *blocks += (unsigned)(fillBlocks > 0 ? fillBlocks : 1);
  return fill;
}

// Calls f(constant) for 1, 2, 4 or 8.
template <typename F> bool withPer(int per, F &&f) {
  if (per == 1)
    return f(std::integral_constant<int, 1>());
  if (per == 2)
    return f(std::integral_constant<int, 2>());
  if (per == 4)
    return f(std::integral_constant<int, 4>());
  return f(std::integral_constant<int, 8>());
}

} // namespace

namespace nmb {
namespace rows {

// Two (key, entry) buffers, the counts and the digits' totals.  A sort of several
// passes whose caller does not ask for the sorted keys keeps them in the first
// buffer, for the offsets.
size_t sortBytes(int64_t count, int64_t groups) {
  const size_t pairs = padded((size_t)count * 4);
  if (isFew(count, groups))
    return groups > kFewGroups ? pairs : 0; // the sorted keys, for the offsets
  const size_t blocks = (size_t)manyBlocks(count), passes = (size_t)passesOf(groups);
  return 4 * pairs + passes * countBytes(blocks) + (blocks > kMostBlocks ? padded((blocks + 1) * kBins * 4) : 0);
}

bool sortByKey(const Stream &s, const char *who, const GPUXIndex &ids, int64_t groups, int32_t *order,
               uint32_t *keys, int32_t *place, int32_t *offsets, void *workspace, uint32_t *words,
               int64_t wordCount, Clearing *clearing) {
  const int64_t n = ids.count;
  const Ids in{ids.data, ids.bytes, (uint32_t)groups};
  const int bits = bitsOf(groups), passes = passesOf(groups);
  const unsigned offsetBlocks = (unsigned)((groups + kOffsetThreads) / kOffsetThreads);
  if (n == 0) {
    if (!offsets)
      return true;
    nmb_sort_nothing<<<offsetBlocks, kOffsetThreads, 0, s.stream>>>(groups, offsets);
    return launched(who);
  }
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  const size_t pairs = padded((size_t)n * 4);
  const bool offsetsApart = isFew(n, groups) ? groups > kFewGroups : passes > 1;
  if (offsetsApart && offsets && !keys)
    keys = reinterpret_cast<uint32_t *>(ws); // the sorted keys, wanted for the offsets below
  if (isFew(n, groups)) {
    // a warp per entry, and for every few of the offsets
    const int64_t warps = offsets && groups <= kFewGroups && groups / 4 > n ? groups / 4 : n;
    const int blocks = (int)((warps + kFewWarps - 1) / kFewWarps);
    unsigned grid;
    const Fill fill = takeRows(clearing, blocks, &grid);
    nmb_sort_few<<<grid, kFewThreads, 0, s.stream>>>(
        in, (int)n, blocks, Results{order, keys, place, groups <= kFewGroups ? offsets : nullptr},
        Clear{words, wordCount}, fill);
    if (!launched(who))
      return false;
  } else {
    const int64_t blocks = manyBlocks(n);
    uint32_t *keyBuf[2] = {reinterpret_cast<uint32_t *>(ws), reinterpret_cast<uint32_t *>(ws + pairs)};
    int32_t *entryBuf[2] = {reinterpret_cast<int32_t *>(ws + 2 * pairs), reinterpret_cast<int32_t *>(ws + 3 * pairs)};
    const size_t countSize = countBytes((size_t)blocks);
    // the counts of each pass in memory of their own, one behind the other
    const int digitBits = (bits + passes - 1) / passes, bins = 1 << digitBits;
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + 4 * pairs);
    const int64_t countWords = blocks * (bins / 2);
    uint32_t *added = blocks > kMostBlocks
                          ? reinterpret_cast<uint32_t *>(ws + 4 * pairs + (size_t)passes * countSize)
                          : nullptr;
    Pass p{in, nullptr, nullptr, counts, nullptr, added, n, (int)blocks, 0, bins, digitBits};
    const bool ok = withPer(perThread(n), [&](auto P) {
      static std::atomic<bool> ready[64];
      if (!nmb::rows::allowShared(who, nmb_sort_scatter<P.value>, kScatterBytes, ready, s.device))
        return false;
      unsigned grid;
      const Fill beside = takeRows(clearing, (int)blocks, &grid);
      nmb_sort_count<P.value><<<grid, kThreads, 0, s.stream>>>(
          p, Clear{counts + countWords, (passes - 1) * countWords}, Clear{words, wordCount}, beside);
      if (!launched(who))
        return false;
      for (int pass = 0; pass < passes; ++pass) {
        const bool last = pass + 1 == passes;
        // the passes alternate between the buffers so that the last one may write
        // sorted keys into buffer 0 (see above)
        const int to = (passes - 1 - pass) & 1;
        p.shift = pass * digitBits;
        p.counts = counts + pass * countWords;
        p.next = last ? nullptr : p.counts + countWords;
        if (added) {
          nmb_sort_add<<<(unsigned)((bins + kAddThreads / 32 - 1) / (kAddThreads / 32)), kAddThreads, 0, s.stream>>>(p);
          if (!launched(who))
            return false;
        }
        const Fill fill = takeRows(clearing, (int)blocks, &grid);
        launchBehind(nmb_sort_scatter<P.value>, grid, kThreads, kScatterBytes, s.stream, true, p, last ? keys : keyBuf[to],
                     last ? order : entryBuf[to], last ? place : nullptr, passes == 1 ? offsets : nullptr, fill);
        if (!launched(who))
          return false;
        p.keysIn = keyBuf[to];
        p.entriesIn = entryBuf[to];
      }
      return true;
    });
    if (!ok)
      return false;
  }
  if (offsets && offsetsApart) {
    nmb_sort_offsets<<<offsetBlocks, kOffsetThreads, 0, s.stream>>>(keys, n, groups, offsets);
    return launched(who);
  }
  return true;
}

} // namespace rows
} // namespace nmb

GPUX_EXPORT size_t _mlir_ciface_nmb_group_rows_workspace(int64_t count, int64_t groups) {
  const int64_t most = 0x7fffffff; // what the entry takes
  return count < 0 || count > most || groups < 0 || groups >= most ? 0 : nmb::rows::sortBytes(count, groups);
}

GPUX_EXPORT int _mlir_ciface_nmb_group_rows_device(void *queue, const GPUXIndex *ids, int64_t groups, int32_t *order,
                                                   int32_t *place, int32_t *offsets, void *workspace,
                                                   size_t workspaceBytes) {
  const char *who = "group_rows";
  if (!nmb::rows::checkIndex(who, ids) || !nmb::rows::checkGroups(who, ids, groups, order, place, offsets))
    return 1;
  nmb::rows::Stream s(queue);
  if (!s.ok)
    return 1;
  nmb::rows::Workspace ws(s, who, workspace, workspaceBytes, nmb::rows::sortBytes(ids->count, groups));
  if (!ws.ok)
    return 1;
  return nmb::rows::sortByKey(s, who, *ids, groups, order, nullptr, place, offsets, ws.data) ? 0 : 1;
}
