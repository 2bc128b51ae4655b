// Eviction from a paged cache: of each request that is over its budget, every kv head
// keeps the newest tokens and, of the others, those of the largest accumulated weights
// (fa_weights.hip), in their order at the front of its pages. No counterpart in the
// reference, which has no cache.
//
// Two launches. evict_select_kernel, a workgroup per request and kv head, finds the
// least weight that is kept by its bits, eight at a time from the highest (a histogram
// of the weights that agree with it so far), then lists the kept tokens in order and
// moves their weights. evict_move_kernel moves the rows by that list, a workgroup per
// request, kv head, pool and slice of a row.
//
// Rows move in place. Kept token number r comes from a token i >= r, so tiles of rows in
// order are safe: a tile's rows are all read before they are written, and what it writes
// lies at or before what it read, below all that the tiles behind it read.
#include <algorithm>

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kPer = 4;     // tokens in a row that a thread lists
constexpr int kCopies = 32;  // of the histogram, by lane: their banks differ

// Weights as whole numbers in their order: NaN above all, both zeros alike.
__device__ __forceinline__ uint32_t order_of(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// A request's lengths, and what its kv heads keep: `heavy` of the first `old` tokens,
// and those from there on.
struct Budget {
  int len, kept, old, heavy;
  __device__ __forceinline__ Budget(const EvictArgs& a, int b) {
    len = min(max(a.kv_len[b], 0), a.table_width << a.pool.page_shift);
    kept = min(len, max(a.max_len[b], 0));
    const int newest = min(a.recent, kept);
    old = len - newest;
    heavy = kept - newest;
  }
  __device__ __forceinline__ bool over() const { return kept < len; }
};

// The workspace of a request's kv head: the first kept token that moves, then the tokens
// that are kept.
__device__ __forceinline__ int* kept_of(const EvictArgs& a, int head) {
  return a.kept + (size_t)head * ((size_t)(a.table_width << a.pool.page_shift) + 1);
}

struct Table {
  const int* table;
  int shift, mask, pages;
  __device__ __forceinline__ Table(const EvictArgs& a, int b)
      : table(a.table + b * a.table_stride), shift(a.pool.page_shift),
        mask((1 << a.pool.page_shift) - 1), pages(a.pool.pages) {}
  // A token's page, -1 where that is outside the pool.
  __device__ __forceinline__ int page(int i) const {
    const int p = table[i >> shift];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
};

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256 * kCopies];
  __shared__ int waves[kSelWaves];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x - b * a.Hkv;
  const Budget q(a, b);
  if (h == 0 && tid == 0) a.new_len[b] = q.kept;
  if (!q.over()) return;
  const Table table(a, b);
  float* const weights = a.weights.w + h * a.weights.head_stride;
  auto weight_at = [&](int i, int page) {
    return weights + page * a.weights.page_stride + (i & table.mask) * a.weights.row_stride;
  };
  // (tokens in pages outside the pool weigh less than any other)
  auto key_at = [&](int i) {
    const int page = table.page(i);
    return page < 0 ? 0u : order_of(*weight_at(i, page));
  };

  // The heavy-th largest key: its high bits so far, and how many of the keys that
  // agree with them are kept.
  uint32_t high = 0;
  int left = q.heavy;
  for (int shift = 24; shift >= 0 && q.heavy > 0; shift -= 8) {
    for (int x = tid; x < 256 * kCopies; x += kSelThreads) hist[x] = 0;
    __syncthreads();
    for (int i = tid; i < q.old; i += kSelThreads) {
      const uint32_t key = key_at(i);
      if (shift == 24 || key >> (shift + 8) == high >> (shift + 8))
        atomicAdd(&hist[(key >> shift & 255) * kCopies + (lane & (kCopies - 1))], 1);
    }
    __syncthreads();
    // Wave w sums bins 16 w .. 16 w + 15, four lanes to a bin.
    const int bin = tid >> 2;
    int sum = 0;
    for (int x = tid & 3; x < kCopies; x += 4) sum += hist[bin * kCopies + x];
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    __syncthreads();
    if ((tid & 3) == 0) hist[bin] = sum;
    __syncthreads();
    if (wave == 0) {  // from the highest bin down, four to a lane
      int mine = 0;
      for (int x = 0; x < 4; ++x) mine += hist[255 - 4 * lane - x];
      int above = wave_prefix(mine, [](int x, int y) { return x + y; }) - mine;
      if (above < left && above + mine >= left) {
        for (int x = 0; x < 4; ++x) {
          const int n = hist[255 - 4 * lane - x];
          if (above + n >= left) {
            found[0] = 255 - 4 * lane - x;
            found[1] = left - above;
            break;
          }
          above += n;
        }
      }
    }
    __syncthreads();
    high |= (uint32_t)found[0] << shift;
    left = found[1];
    __syncthreads();
  }

  // The kept tokens in order: those above `high`, the first `left` of those equal to it,
  // and the newest.
  int* const kept = kept_of(a, blockIdx.x);
  int above = 0, equal = 0;  // of the chunks before
  for (int i0 = 0; i0 < q.len; i0 += kSelThreads * kPer) {
    const int i = i0 + tid * kPer;
    float w[kPer];
    int counts = 0;      // above in the low half, equal in the high one
    uint32_t flags = 0;  // above, equal, and in no page, a bit each in its byte
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      w[x] = 0.f;
      if (i + x >= q.len) continue;
      const int page = table.page(i + x);
      if (page >= 0) w[x] = *weight_at(i + x, page);
      else flags |= 65536u << x;
      if (i + x >= q.old) {
        counts += 1;
        flags |= 1u << x;
      } else if (q.heavy > 0) {
        const uint32_t key = page < 0 ? 0u : order_of(w[x]);
        if (key > high) {
          counts += 1;
          flags |= 1u << x;
        } else if (key == high) {
          counts += 1 << 16;
          flags |= 256u << x;
        }
      }
    }
    const int upto = wave_prefix(counts, [](int x, int y) { return x + y; });
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int before = upto - counts, all = 0;
    for (int x = 0; x < kSelWaves; ++x) {
      before += x < wave ? waves[x] : 0;
      all += waves[x];
    }
    int n_above = above + (before & 0xffff), n_equal = equal + (int)((unsigned)before >> 16);
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const bool is_above = flags >> x & 1, is_equal = flags >> (8 + x) & 1;
      const int r = n_above + min(n_equal, left);
      if (is_above || (is_equal && n_equal < left)) {
        kept[1 + r] = i + x;
        if (r < i + x && !(flags >> (16 + x) & 1)) {
          const int page = table.page(r);
          if (page >= 0) *weight_at(r, page) = w[x];
        }
      } else if (i + x < q.len && r == i + x) {
        kept[0] = r;  // (the first that is not kept: all before it are)
      }
      n_above += is_above;
      n_equal += is_equal;
    }
    above += all & 0xffff;
    equal += (int)((unsigned)all >> 16);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256, kMoveRows = 8;  // rows of a tile that a thread moves
constexpr int kSlice = 128;                       // bytes of a row that a workgroup moves

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictArgs a, int slices) {
  const int head = blockIdx.x, b = head / a.Hkv, h = head - b * a.Hkv;
  const Budget q(a, b);
  if (!q.over()) return;
  const int* const kept = kept_of(a, head);
  const int first = kept[0];
  const Table table(a, b);
  const int part = blockIdx.y, tid = threadIdx.x;
  if (part < 2 * slices) {  // a slice of K's or V's rows
    uint8_t* const pool =
        (uint8_t*)(part < slices ? a.pool.k : a.pool.v) + h * a.pool.head_stride + part % slices * kSlice;
    const int bytes = min(kSlice, a.row_bytes - part % slices * kSlice);
    constexpr int kLanes = kSlice / 16, kAtOnce = kMoveThreads / kLanes;  // rows at once
    const int col = 16 * (tid % kLanes);
    auto row_of = [&](int i) -> uint8_t* {
      const int page = table.page(i);
      return page < 0 || col >= bytes ? nullptr
                                      : pool + page * a.pool.page_stride + (i & table.mask) * a.pool.row_stride + col;
    };
    for (int r0 = first; r0 < q.kept; r0 += kAtOnce * kMoveRows) {
      u32x4 x[kMoveRows];
      uint32_t there = 0;  // rows that have a page
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        const int r = r0 + e * kAtOnce + tid / kLanes;
        const uint8_t* from = r < q.kept ? row_of(kept[1 + r]) : nullptr;
        x[e] = from ? *reinterpret_cast<const u32x4*>(from) : u32x4{0u, 0u, 0u, 0u};
        there |= (from ? 1u : 0u) << e;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        const int r = r0 + e * kAtOnce + tid / kLanes;
        uint8_t* to = there >> e & 1 ? row_of(r) : nullptr;
        if (to) *reinterpret_cast<u32x4*>(to) = x[e];
      }
    }
    return;
  }
  // The scales of K's or V's rows, a row per thread.
  uint8_t* const scales = (part == 2 * slices ? a.scales.k : a.scales.v) + h * a.scales.head_stride;
  auto scale_of = [&](int i) -> uint8_t* {
    const int page = table.page(i);
    return page < 0 ? nullptr : scales + page * a.scales.page_stride + (i & table.mask) * a.scales.row_stride;
  };
  for (int r0 = first; r0 < q.kept; r0 += kMoveThreads) {
    const int r = r0 + tid;
    const uint8_t* from = r < q.kept ? scale_of(kept[1 + r]) : nullptr;
    uint8_t x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from && e < a.scale_bytes ? from[e] : 0;
    __syncthreads();
    uint8_t* to = from ? scale_of(r) : nullptr;
    if (to)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < a.scale_bytes) to[e] = x[e];
  }
}

}  // namespace

size_t evict_workspace_bytes(int B, int Hkv, int table_width, int page_size) {
  return (size_t)B * Hkv * ((size_t)table_width * page_size + 1) * sizeof(int);
}

hipError_t launch_paged_evict(const EvictArgs& a, void* stream) {
  const unsigned heads = (unsigned)(a.B * a.Hkv);
  hipLaunchKernelGGL(evict_select_kernel, dim3(heads), dim3(kSelThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int slices = (a.row_bytes + kSlice - 1) / kSlice;
  hipLaunchKernelGGL(evict_move_kernel, dim3(heads, (unsigned)(2 * slices + (a.scales.k ? 2 : 0))),
                     dim3(kMoveThreads), 0, (hipStream_t)stream, a, slices);
  return hipGetLastError();
}

}  // namespace fa
