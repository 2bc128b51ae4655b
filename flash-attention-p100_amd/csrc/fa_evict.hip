// Eviction from a paged cache: of each request that is over its budget, every kv head
// keeps the newest tokens and, of the others, those of the largest accumulated weights
// (fa_weights.hip), in their order at the front of its pages. No counterpart in the
// reference, which has no cache.
//
// Three launches. evict_select_kernel, a workgroup per request and kv head, finds the
// least weight that is kept by its bits, eight at a time from the highest (a histogram
// of the weights that agree with it so far), then lists the kept tokens in order and
// moves their weights. The rows then move by that list in two:
//   * tokens from within the kept length L move in place, by a workgroup per request, kv
//     head, pool and slice of a row. Kept token number r comes from a token i >= r, so
//     tiles of rows in order are safe: a tile's rows are all read before they are
//     written, and what it writes lies at or before what it read, below all that the
//     tiles behind it read;
//   * tokens from behind L: nothing writes there, and what their places held has moved,
//     so all of them move at once.
// Bound by HBM where many rows move (evict_inner_kernel 55 us for 32 requests of 8
// kv heads of 1024 rows of 128, 268 MB read and written), else by latency.
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

// The workspace of a request's kv head: the number of the first kept token that moves and
// of the first from behind the kept length, then the tokens that are kept.
constexpr int kHead = 2;
__device__ __forceinline__ int* kept_of(const EvictArgs& a, int head) {
  return a.kept + (size_t)head * ((size_t)(a.table_width << a.pool.page_shift) + kHead);
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

// HOLD: up to kHeld tokens, whose weights are read once and stay in registers.
constexpr int kHeldChunks = 8, kChunk = kSelThreads * kPer, kHeld = kHeldChunks * kChunk;
template <bool HOLD>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256 * kCopies];
  __shared__ int waves[2][kSelWaves];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x - b * a.Hkv;
  const Budget q(a, b);
  if (HOLD && h == 0 && tid == 0) a.new_len[b] = q.kept;
  if (!q.over() || (q.len <= kHeld) != HOLD) return;  // (the other launch's)
  const Table table(a, b);
  float* const weights = a.weights.w + h * a.weights.head_stride;
  // The weights of tokens i .. i + kPer - 1, and which of them have a page.
  struct Four {
    float w[kPer];
    uint32_t there;
  };
  auto read = [&](int i) {
    Four x;
    x.there = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      x.w[e] = 0.f;
      if (i + e >= q.len) continue;
      const int page = table.page(i + e);
      if (page < 0) continue;
      x.w[e] = weights[page * a.weights.page_stride + ((i + e) & table.mask) * a.weights.row_stride];
      x.there |= 1u << e;
    }
    return x;
  };
  // (tokens in pages outside the pool weigh less than any other)
  auto key_of = [&](const Four& x, int e) { return x.there >> e & 1 ? order_of(x.w[e]) : 0u; };
  constexpr int kHere = HOLD ? kHeldChunks : 1;
  Four held[kHere];
  if constexpr (HOLD) {
#pragma unroll
    for (int c = 0; c < kHere; ++c) held[c] = read(c * kChunk + tid * kPer);
  }
  // do_chunk(first token, this thread's weights) over all chunks of `n` tokens.
  auto chunks = [&](int n, auto&& do_chunk) {
    if constexpr (HOLD) {
#pragma unroll
      for (int c = 0; c < kHere; ++c)
        if (c * kChunk < n) do_chunk(c * kChunk + tid * kPer, held[c]);
    } else {
      for (int i0 = 0; i0 < n; i0 += kChunk) do_chunk(i0 + tid * kPer, read(i0 + tid * kPer));
    }
  };

  // The heavy-th largest key: its high bits so far, and how many of the keys that
  // agree with them are kept.
  uint32_t high = 0;
  int left = q.heavy;
  for (int shift = 24; shift >= 0 && q.heavy > 0; shift -= 8) {
    for (int x = tid; x < 256 * kCopies; x += kSelThreads) hist[x] = 0;
    __syncthreads();
    chunks(q.old, [&](int i, const Four& x) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t key = key_of(x, e);
        if (i + e < q.old && (shift == 24 || key >> (shift + 8) == high >> (shift + 8)))
          atomicAdd(&hist[(key >> shift & 255) * kCopies + (lane & (kCopies - 1))], 1);
      }
    });
    __syncthreads();
    // Four threads to a bin, neighbours at neighbouring copies.
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
  // and the newest. A chunk's weights are all read before any is written (into places at or
  // before their own, which no chunk behind reads).
  int* const kept = kept_of(a, blockIdx.x);
  int above = 0, equal = 0, turn = 0;  // of the chunks before
  chunks(q.len, [&](int i, const Four& four) {
    int counts = 0;      // above in the low half, equal in the high one
    uint32_t flags = 0;  // above and equal, a bit each in its byte
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      if (i + x >= q.len) continue;
      if (i + x >= q.old) {
        counts += 1;
        flags |= 1u << x;
      } else if (q.heavy > 0) {
        const uint32_t key = key_of(four, x);
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
    if (lane == 63) waves[turn][wave] = upto;
    __syncthreads();
    int before = upto - counts, all = 0;
    for (int x = 0; x < kSelWaves; ++x) {
      before += x < wave ? waves[turn][x] : 0;
      all += waves[turn][x];
    }
    int n_above = above + (before & 0xffff), n_equal = equal + (int)((unsigned)before >> 16);
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const bool is_above = flags >> x & 1, is_equal = flags >> (8 + x) & 1;
      const int r = n_above + min(n_equal, left);
      if (i + x == q.kept) kept[1] = r;
      if (is_above || (is_equal && n_equal < left)) {
        kept[kHead + r] = i + x;
        if (r < i + x && (four.there >> x & 1)) {
          const int page = table.page(r);
          if (page >= 0)
            weights[page * a.weights.page_stride + (r & table.mask) * a.weights.row_stride] = four.w[x];
        }
      } else if (i + x < q.len && r == i + x) {
        kept[0] = r;  // (the first that is not kept: all before it are)
      }
      n_above += is_above;
      n_equal += is_equal;
    }
    above += all & 0xffff;
    equal += (int)((unsigned)all >> 16);
    turn ^= 1;
  });
}

// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 512, kMoveRows = 8;  // rows of a tile that a thread moves
constexpr int kSlice = 128;                       // bytes of a row that a workgroup moves

// A kv head's rows of one pool, as units of 16 bytes from column `col` on; null where a
// token has no page.
struct Rows {
  uint8_t* pool;
  long long page_stride, row_stride;
  Table table;
  __device__ __forceinline__ Rows(const EvictArgs& a, int b, int h, bool v, int col)
      : pool((uint8_t*)(v ? a.pool.v : a.pool.k) + h * a.pool.head_stride + col),
        page_stride(a.pool.page_stride), row_stride(a.pool.row_stride), table(a, b) {}
  __device__ __forceinline__ uint8_t* at(int i) const {
    const int page = table.page(i);
    return page < 0 ? nullptr : pool + page * page_stride + (i & table.mask) * row_stride;
  }
};
struct Scales {
  uint8_t* pool;
  long long page_stride, row_stride;
  Table table;
  __device__ __forceinline__ Scales(const EvictArgs& a, int b, int h, bool v)
      : pool((v ? a.scales.v : a.scales.k) + h * a.scales.head_stride),
        page_stride(a.scales.page_stride), row_stride(a.scales.row_stride), table(a, b) {}
  __device__ __forceinline__ uint8_t* at(int i) const {
    const int page = table.page(i);
    return page < 0 ? nullptr : pool + page * page_stride + (i & table.mask) * row_stride;
  }
};

__global__ __launch_bounds__(kMoveThreads) void evict_inner_kernel(const EvictArgs a, int slices) {
  const int head = blockIdx.x, b = head / a.Hkv, h = head - b * a.Hkv;
  const Budget q(a, b);
  if (!q.over()) return;
  const int* const kept = kept_of(a, head);
  const int first = kept[0], end = kept[1];
  const int part = blockIdx.y, tid = threadIdx.x;
  if (part < 2 * slices) {  // a slice of K's or V's rows
    const int slice = part % slices * kSlice, bytes = min(kSlice, a.row_bytes - slice);
    constexpr int kLanes = kSlice / 16, kAtOnce = kMoveThreads / kLanes;  // rows at once
    const int col = 16 * (tid % kLanes);
    const Rows rows(a, b, h, part >= slices, slice + col);
    for (int r0 = first; r0 < end; r0 += kAtOnce * kMoveRows) {
      u32x4 x[kMoveRows];
      uint32_t there = 0;  // rows that have a page
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        const int r = r0 + e * kAtOnce + tid / kLanes;
        const uint8_t* from = r < end && col < bytes ? rows.at(kept[kHead + r]) : nullptr;
        x[e] = from ? *reinterpret_cast<const u32x4*>(from) : u32x4{0u, 0u, 0u, 0u};
        there |= (from ? 1u : 0u) << e;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        uint8_t* to = there >> e & 1 ? rows.at(r0 + e * kAtOnce + tid / kLanes) : nullptr;
        if (to) *reinterpret_cast<u32x4*>(to) = x[e];
      }
    }
    return;
  }
  // The scales of K's or V's rows, a row per thread.
  const Scales scales(a, b, h, part > 2 * slices);
  for (int r0 = first; r0 < end; r0 += kMoveThreads) {
    const int r = r0 + tid;
    const uint8_t* from = r < end ? scales.at(kept[kHead + r]) : nullptr;
    uint8_t x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from && e < a.scale_bytes ? from[e] : 0;
    __syncthreads();
    uint8_t* to = from ? scales.at(r) : nullptr;
    if (to)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < a.scale_bytes) to[e] = x[e];
  }
}

// A unit of 16 bytes, or a row's scales, at a time; four units in flight.
__global__ __launch_bounds__(256) void evict_outer_kernel(const EvictArgs a) {
  const int head = blockIdx.x, b = head / a.Hkv, h = head - b * a.Hkv;
  const Budget q(a, b);
  if (!q.over()) return;
  const int* const kept = kept_of(a, head);
  const int first = kept[1], n = q.kept - first, units = a.row_bytes / 16;
  const int tid = blockIdx.y * 256 + threadIdx.x, step = gridDim.y * 256;
  constexpr int kAtOnce = 4;
  const long long all = 2LL * n * units;
  for (long long i0 = tid; i0 < all; i0 += (long long)kAtOnce * step) {
    const uint8_t* from[kAtOnce];
    uint8_t* to[kAtOnce];
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const long long i = i0 + (long long)e * step;
      from[e] = to[e] = nullptr;
      if (i >= all) continue;
      const bool v = i >= all / 2;
      const long long x = v ? i - all / 2 : i;
      const int r = (int)(x / units), unit = (int)(x - (long long)r * units);
      const Rows rows(a, b, h, v, 16 * unit);
      from[e] = rows.at(kept[kHead + first + r]);
      to[e] = rows.at(first + r);
    }
    u32x4 x[kAtOnce];
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e)
      if (from[e] && to[e]) x[e] = *reinterpret_cast<const u32x4*>(from[e]);
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e)
      if (from[e] && to[e]) *reinterpret_cast<u32x4*>(to[e]) = x[e];
  }
  if (a.scale_bytes > 0)
    for (long long i = tid; i < 2LL * n; i += step) {
      const bool v = i >= n;
      const int r = (int)(v ? i - n : i);
      const Scales scales(a, b, h, v);
      const uint8_t* from = scales.at(kept[kHead + first + r]);
      uint8_t* to = scales.at(first + r);
      if (from && to)
        for (int e = 0; e < a.scale_bytes; ++e) to[e] = from[e];
    }
}

}  // namespace

size_t evict_workspace_bytes(int B, int Hkv, int table_width, int page_size) {
  return (size_t)B * Hkv * ((size_t)table_width * page_size + kHead) * sizeof(int);
}

hipError_t launch_paged_evict(const EvictArgs& a, void* stream) {
  const unsigned heads = (unsigned)(a.B * a.Hkv);
  const long long cap = (long long)a.table_width << a.pool.page_shift;
  hipLaunchKernelGGL(evict_select_kernel<true>, dim3(heads), dim3(kSelThreads), 0, (hipStream_t)stream, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && cap > kHeld) {  // (requests of more tokens, if there are any)
    hipLaunchKernelGGL(evict_select_kernel<false>, dim3(heads), dim3(kSelThreads), 0, (hipStream_t)stream, a);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const int slices = (a.row_bytes + kSlice - 1) / kSlice;
  hipLaunchKernelGGL(evict_inner_kernel, dim3(heads, (unsigned)(2 * slices + (a.scales.k ? 2 : 0))),
                     dim3(kMoveThreads), 0, (hipStream_t)stream, a, slices);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // (at least four workgroups to a CU, as far as there can be that many units)
  const long long most = (2 * cap * (a.row_bytes / 16) + 1023) / 1024;
  const unsigned per_head = (unsigned)std::max(1LL, std::min<long long>((4LL * kCUs + heads - 1) / heads, most));
  hipLaunchKernelGGL(evict_outer_kernel, dim3(heads, per_head), dim3(256), 0, (hipStream_t)stream, a);
  return hipGetLastError();
}

}  // namespace fa
