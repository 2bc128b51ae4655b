// Eviction from a paged cache: of each request that is over its budget, every kv head
// keeps the newest tokens and, of the others, those of the largest accumulated weights
// (fa_weights.hip), in their order at the front of its pages. No counterpart in the
// reference, which has no cache.
//
// evict_select_kernel, a workgroup per request and kv head, finds the least weight that is
// kept by its bits, eight at a time from the highest (a histogram of the weights that agree
// with it so far), then lists the kept tokens in order. Their rows, scales and weights then
// move by that list. Kept token number r comes from a token i >= r, so tiles of rows in
// order are safe: a tile's rows are all read before they are written, and what it writes
// lies at or before what it read, below all that the tiles behind it read. Where there is a
// kv head for every CU, or little to move, the same workgroup goes over the tiles; else two
// more launches take what workgroups can share:
//   * tokens from within the kept length L, by a workgroup per pool and slice of a row;
//   * tokens from behind L: nothing writes there, and what their places held has moved,
//     so all of them move at once.
// Bound by HBM where many rows move: 32 requests of 8 kv heads of 1100 rows of 256 bytes of
// which 1024 stay, 270 MB read and written, take 54 us, 10 of them selecting (in 4 bits, 71
// MB: 22 us); 4 requests of 16384 to 32768 tokens of which 4096 stay, 28 us of selecting
// (half of that reading 3 MB of weights and counting: one CU to a kv head) and 12 + 43 us of
// moving 134 MB (in 4 bits, 36 MB: 27, 10 + 26).
#include <algorithm>

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kPer = 4;     // tokens in a row that a thread lists
constexpr int kCopies = 32;  // of the histogram, by lane: their banks differ

// Weights as whole numbers in their order: NaN above all others, both zeros alike. None is 0
// or kNewest.
constexpr uint32_t kNewest = 0xffffffffu;
__device__ __forceinline__ uint32_t order_of(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return kNewest - 1;
  if (u == 0x80000000u) u = 0;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// A request's lengths, and how many of the newest tokens stay.
struct Budget {
  int len, kept, newest;
  __device__ __forceinline__ Budget(const EvictArgs& a, int b) {
    len = min(max(a.kv_len[b], 0), a.table_width << a.pool.page_shift);
    kept = min(len, max(a.max_len[b], 0));
    newest = min(a.recent, kept);
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

// HOLD: up to kHeld tokens, whose keys are made once and stay in registers, 32 a thread. Of
// longer requests weights are read again for each of the four digits and for the list, a
// chunk at a time: two kv heads of 32768 tokens are selected in 26 us, of 33000 in 50, of
// 65536 in 84, of 131072 in 166. (More registers, or several chunks in flight there: not tried.)
constexpr int kHeldChunks = 8, kChunk = kSelThreads * kPer, kHeld = kHeldChunks * kChunk;
struct SelectLds {
  __attribute__((aligned(16))) int hist[256 * kCopies];
  __attribute__((aligned(16))) int bins[2][256];
  int waves[2][kHeldChunks][kSelWaves];
};
template <bool HOLD>
__device__ __forceinline__ void select(const EvictArgs& a, const Budget& q, int b, int h, SelectLds& lds) {
  constexpr int kHere = HOLD ? kHeldChunks : 1;  // chunks at once
  auto& [hist, bins, waves] = lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Table table(a, b);
  const float* const weights = a.weights.w + h * a.weights.head_stride;
  // The keys of tokens i .. i + kPer - 1, by which the `kept` largest stay: the newest tokens'
  // are above all weights, those of tokens outside the pool and behind the request (of equal
  // keys the first stay, so none of these does) below.
  struct Four {
    uint32_t key[kPer];
  };
  // Four tokens lie together: 32768 of them are read in 8 us instead of 16.
  const bool wide = a.weights.row_stride == 1 && table.shift >= 2 &&
                    (((uintptr_t)weights & 15) | ((4 * a.weights.page_stride) & 15)) == 0;
  struct Pages {
    int of[kPer];
  };
  auto read_pages = [&](int i) {
    Pages x;
    if (wide) {
      x.of[0] = table.page(min(i, q.len - 1));
      return x;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) x.of[e] = table.page(min(i + e, q.len - 1));
    return x;
  };
  auto read = [&](int i, const Pages& pages) {
    floatx4 w;
    bool there[kPer];
    if (wide) {
      const int row = min(i, (q.len - 1) & -kPer) & table.mask;
      w = *reinterpret_cast<const floatx4*>(weights + max(pages.of[0], 0) * a.weights.page_stride + row);
#pragma unroll
      for (int e = 0; e < kPer; ++e) there[e] = pages.of[0] >= 0;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int row = min(i + e, q.len - 1) & table.mask;
        w[e] = weights[max(pages.of[e], 0) * a.weights.page_stride + row * a.weights.row_stride];
        there[e] = pages.of[e] >= 0;
      }
    }
    Four x;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float one = w[e];
      x.key[e] = there[e] ? order_of(one) : 0u;
      if (i + e >= q.len - q.newest) x.key[e] = i + e < q.len ? kNewest : 0u;
    }
    return x;
  };
  Four held[kHere];
  if constexpr (HOLD) {
    // (all pages, then all weights, without a branch around a thread's own: one wait each.
    // Token by token, 20 us of the 60 that 32768 tokens took.)
    Pages pages[kHere];
#pragma unroll
    for (int c = 0; c < kHere; ++c)
      if (c * kChunk < q.len) pages[c] = read_pages(c * kChunk + tid * kPer);
#pragma unroll
    for (int c = 0; c < kHere; ++c)
      if (c * kChunk < q.len) held[c] = read(c * kChunk + tid * kPer, pages[c]);
  }

  // The kept-th largest key: its high bits so far, and how many of the keys that agree with
  // them stay. (None does where nothing is kept.)
  uint32_t high = q.kept > 0 ? 0u : kNewest;
  int left = q.kept;
  const u32x4 zeros = {0u, 0u, 0u, 0u};
  if (left > 0) {
    for (int x = tid; x < 256 * kCopies / 4; x += kSelThreads) reinterpret_cast<u32x4*>(hist)[x] = zeros;
    __syncthreads();
  }
  for (int shift = 24; shift >= 0 && q.kept > 0; shift -= 8) {
    const uint32_t agree = shift == 24 ? 0u : ~0u << (shift + 8);
    auto count = [&](const Four& x) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if ((x.key[e] & agree) == high)
          atomicAdd(&hist[(x.key[e] >> shift & 255) * kCopies + (lane & (kCopies - 1))], 1);
    };
    if constexpr (HOLD) {
#pragma unroll
      for (int c = 0; c < kHere; ++c)
        if (c * kChunk < q.len) count(held[c]);
    } else {
      for (int i = tid * kPer; i < q.len + tid * kPer; i += kChunk) count(read(i, read_pages(i)));
    }
    __syncthreads();
    // Four threads to a bin, each with two of its eight units of four copies (by places whose
    // banks differ), which are cleared again.
    const int bin = tid >> 2;
    int sum = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int place = ((tid & 3) + 4 * x + 2 * (bin & 2)) & 7;
      u32x4& unit = reinterpret_cast<u32x4*>(hist)[bin * (kCopies / 4) + place];
      const u32x4 n = unit;
      unit = zeros;
      sum += n[0] + n[1] + n[2] + n[3];
    }
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    if ((tid & 3) == 0) bins[shift >> 3 & 1][bin] = sum;
    __syncthreads();
    // Each wave goes through them from the highest down, four to a lane.
    const u32x4 n = reinterpret_cast<const u32x4*>(bins[shift >> 3 & 1])[63 - lane];
    const int mine = n[0] + n[1] + n[2] + n[3];
    int above = wave_prefix(mine, [](int x, int y) { return x + y; }) - mine;
    const int at = __ffsll(__ballot(above < left && above + mine >= left)) - 1;
    int bin_at = 255 - 4 * lane;
#pragma unroll
    for (int x = 0; x < 3; ++x)
      if (bin_at == 255 - 4 * lane - x && above + (int)n[3 - x] < left) {
        above += n[3 - x];
        --bin_at;
      }
    high |= (uint32_t)__builtin_amdgcn_readlane(bin_at, at) << shift;
    left -= __builtin_amdgcn_readlane(above, at);
  }

  // The kept tokens in order: those above `high` and the first `left` of those equal to it.
  int* const kept = kept_of(a, blockIdx.x);
  int above = 0, equal = 0, turn = 0;  // of the chunks before
  for (int i0 = 0; i0 < q.len; i0 += kHere * kChunk) {
    Four keys[kHere];
    int counts[kHere], upto[kHere];  // above in the low half, equal in the high one
#pragma unroll
    for (int c = 0; c < kHere; ++c) {
      counts[c] = 0;
      const int i = i0 + c * kChunk + tid * kPer;
      if (i0 + c * kChunk < q.len) {
        if constexpr (HOLD)
          keys[c] = held[c];
        else
          keys[c] = read(i, read_pages(i));
#pragma unroll
        for (int x = 0; x < kPer; ++x)
          counts[c] += keys[c].key[x] > high ? 1 : keys[c].key[x] == high ? 1 << 16 : 0;
        upto[c] = wave_prefix(counts[c], [](int x, int y) { return x + y; });
        if (lane == 63) waves[turn][c][wave] = upto[c];
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kHere; ++c) {
      if (i0 + c * kChunk >= q.len) break;
      const int sums = wave_prefix(waves[turn][c][lane & (kSelWaves - 1)], [](int x, int y) { return x + y; });
      const int before = upto[c] - counts[c] + (wave > 0 ? __builtin_amdgcn_readlane(sums, wave - 1) : 0);
      const int all = __builtin_amdgcn_readlane(sums, kSelWaves - 1);
      int n_above = above + (before & 0xffff), n_equal = equal + (int)((unsigned)before >> 16);
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int i = i0 + c * kChunk + tid * kPer + x;
        const bool is_above = keys[c].key[x] > high, is_equal = keys[c].key[x] == high;
        const int r = n_above + min(n_equal, left);
        if (i == q.kept) kept[1] = r;
        if (is_above || (is_equal && n_equal < left))
          kept[kHead + r] = i;
        else if (r == i)
          kept[0] = r;  // (the first that does not stay: all before it do)
        n_above += is_above;
        n_equal += is_equal;
      }
      above += all & 0xffff;
      equal += (int)((unsigned)all >> 16);
    }
    turn ^= 1;
  }
}

// Where a kv head's tokens have something; null where a token has no page.
template <typename T>
struct Places {
  T* first;
  long long page_stride, row_stride;
  Table table;
  __device__ __forceinline__ T* at(int i) const {
    const int page = table.page(i);
    return page < 0 ? nullptr : first + page * page_stride + (i & table.mask) * row_stride;
  }
};
// Their rows of one pool from byte `col` on, their scales of one, their weights.
__device__ __forceinline__ Places<uint8_t> rows_of(const EvictArgs& a, int b, int h, bool v, int col) {
  return {(uint8_t*)(v ? a.pool.v : a.pool.k) + h * a.pool.head_stride + col, a.pool.page_stride,
          a.pool.row_stride, Table(a, b)};
}
__device__ __forceinline__ Places<uint8_t> scales_of(const EvictArgs& a, int b, int h, bool v) {
  return {(v ? a.scales.v : a.scales.k) + h * a.scales.head_stride, a.scales.page_stride, a.scales.row_stride,
          Table(a, b)};
}
__device__ __forceinline__ Places<float> weights_of(const EvictArgs& a, int b, int h) {
  return {a.weights.w + h * a.weights.head_stride, a.weights.page_stride, a.weights.row_stride, Table(a, b)};
}

// What the workgroup's waves have loaded and stored is done: what was read may be written, and
// what was written read. (A barrier alone orders what is issued, and waits for neither.)
__device__ __forceinline__ void all_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Moves a kv head's kept tokens, rows, scales and weights together, tile by tile in order.
// An item is 16 bytes of a row and the scale of its 32 values (both are `lanes` to a row).
constexpr int kItems = 8;  // of a tile that a thread moves
__device__ __forceinline__ void move_all(const EvictArgs& a, int b, int h, int kept_count, const int* kept,
                                         int lanes_log2) {
  const int tid = threadIdx.x, c = tid & ((1 << lanes_log2) - 1), v = tid >> lanes_log2 & 1;
  const int at_once = kSelThreads >> (lanes_log2 + 1), row0 = tid >> (lanes_log2 + 1);
  const auto rows = rows_of(a, b, h, v, 16 * c);
  const auto scales = scales_of(a, b, h, v);
  const auto weights = weights_of(a, b, h);
  const bool live = 16 * c < a.row_bytes, scaled = live && a.scale_bytes > 0, weighed = c == 0 && v == 0;
  for (int r0 = kept[0]; r0 < kept_count; r0 += kItems * at_once) {
    u32x4 x[kItems];
    uint8_t scale[kItems];
    float weight[kItems];
    uint32_t there = 0;
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      const int r = r0 + e * at_once + row0;
      if (r < kept_count && live) {
        const int i = kept[kHead + r];
        const uint8_t* const from = rows.at(i);
        if (from) {
          there |= 1u << e;
          x[e] = *reinterpret_cast<const u32x4*>(from);
          if (scaled) scale[e] = scales.at(i)[c];
          if (weighed) weight[e] = *weights.at(i);
        }
      }
    }
    all_done();
#pragma unroll
    for (int e = 0; e < kItems; ++e) {
      const int r = r0 + e * at_once + row0;
      uint8_t* const to = there >> e & 1 ? rows.at(r) : nullptr;
      if (to) {
        *reinterpret_cast<u32x4*>(to) = x[e];
        if (scaled) scales.at(r)[c] = scale[e];
        if (weighed) *weights.at(r) = weight[e];
      }
    }
  }
}

// ALL: moves them as well.
template <bool ALL>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const EvictArgs a, int lanes_log2) {
  __shared__ SelectLds lds;
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x - b * a.Hkv;
  const Budget q(a, b);
  if (h == 0 && threadIdx.x == 0) a.new_len[b] = q.kept;
  if (!q.over()) return;
  if (q.len <= kHeld)
    select<true>(a, q, b, h, lds);
  else
    select<false>(a, q, b, h, lds);
  if constexpr (ALL) {
    all_done();
    move_all(a, b, h, q.kept, kept_of(a, blockIdx.x), lanes_log2);
  }
}

// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 1024, kMoveRows = 8;  // rows of a tile that a thread moves
// Bytes of a row that a workgroup moves. (4 requests of 8 kv heads that keep 4096 rows of
// 256 bytes, 128 -> 64 -> 32: 53 -> 29 -> 36 us; 32 requests of 1024 rows: 55, 58, 85.)
constexpr int kSlice = 64;

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
    const auto rows = rows_of(a, b, h, part >= slices, slice + col);
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
      all_done();
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        uint8_t* to = there >> e & 1 ? rows.at(r0 + e * kAtOnce + tid / kLanes) : nullptr;
        if (to) *reinterpret_cast<u32x4*>(to) = x[e];
      }
    }
    return;
  }
  if (part == 2 * slices) {  // the weights
    const auto weights = weights_of(a, b, h);
    for (int r0 = first; r0 < end; r0 += kMoveThreads * kMoveRows) {
      float x[kMoveRows];
      uint32_t there = 0;
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        const int r = r0 + e * kMoveThreads + tid;
        const float* from = r < end ? weights.at(kept[kHead + r]) : nullptr;
        x[e] = from ? *from : 0.f;
        there |= (from ? 1u : 0u) << e;
      }
      all_done();
#pragma unroll
      for (int e = 0; e < kMoveRows; ++e) {
        float* to = there >> e & 1 ? weights.at(r0 + e * kMoveThreads + tid) : nullptr;
        if (to) *to = x[e];
      }
    }
    return;
  }
  // The scales of K's or V's rows, a row per thread.
  const auto scales = scales_of(a, b, h, part == 2 * slices + 2);
  for (int r0 = first; r0 < end; r0 += kMoveThreads) {
    const int r = r0 + tid;
    const uint8_t* from = r < end ? scales.at(kept[kHead + r]) : nullptr;
    uint8_t x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from && e < a.scale_bytes ? from[e] : 0;
    all_done();
    uint8_t* to = from ? scales.at(r) : nullptr;
    if (to)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < a.scale_bytes) to[e] = x[e];
  }
}

// Workgroups to a CU. (4 requests of 8 kv heads, 3400 rows of 256 bytes each: 4 -> 16, 41 -> 36 us.)
constexpr int kOuter = 16;
// A unit of 16 bytes, or a row's scales, at a time; four units in flight.
__global__ __launch_bounds__(256) void evict_outer_kernel(const EvictArgs a, int lanes_log2) {
  const int head = blockIdx.x, b = head / a.Hkv, h = head - b * a.Hkv;
  const Budget q(a, b);
  if (!q.over()) return;
  const int* const kept = kept_of(a, head);
  const int first = kept[1], n = q.kept - first;
  const int tid = blockIdx.y * 256 + threadIdx.x, step = gridDim.y * 256;
  constexpr int kAtOnce = 4;
  // (of a number of lanes to a row that is a power of two)
  const long long all = 2LL * n << lanes_log2;
  for (long long i0 = tid; i0 < all; i0 += (long long)kAtOnce * step) {
    const uint8_t* from[kAtOnce];
    uint8_t* to[kAtOnce];
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const long long i = i0 + (long long)e * step;
      from[e] = to[e] = nullptr;
      const int row = (int)(i >> lanes_log2), col = 16 * ((int)i & ((1 << lanes_log2) - 1));
      if (i >= all || col >= a.row_bytes) continue;
      const bool v = row >= n;
      const int r = first + (v ? row - n : row);
      const auto rows = rows_of(a, b, h, v, col);
      from[e] = rows.at(kept[kHead + r]);
      to[e] = rows.at(r);
    }
    u32x4 x[kAtOnce];
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e)
      if (from[e] && to[e]) x[e] = *reinterpret_cast<const u32x4*>(from[e]);
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e)
      if (from[e] && to[e]) *reinterpret_cast<u32x4*>(to[e]) = x[e];
  }
  const auto weights = weights_of(a, b, h);
  for (int r = tid; r < n; r += step) {
    const float* from = weights.at(kept[kHead + first + r]);
    float* to = weights.at(first + r);
    if (from && to) *to = *from;
  }
  if (a.scale_bytes > 0)
    for (long long i = tid; i < 2LL * n; i += step) {
      const bool v = i >= n;
      const int r = (int)(v ? i - n : i);
      const auto scales = scales_of(a, b, h, v);
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
  int lanes_log2 = 0;
  while (16 << lanes_log2 < a.row_bytes) ++lanes_log2;
  // A launch for all where every CU has a kv head, or these are small. (Rows of 256 bytes, us
  // for one launch and for three: 32 requests of 8 heads of up to 1100 tokens 73 and 73, 64 of
  // 2000 151 and 179, 4 of 300 14.6 and 17.4; 16 of 2200 113 and 73, 1 of 2000 22 and 16.)
  const bool all = heads >= (unsigned)kCUs || cap * 2 * a.row_bytes <= 1 << 18;
  const auto select = all ? evict_select_kernel<true> : evict_select_kernel<false>;
  hipLaunchKernelGGL(select, dim3(heads), dim3(kSelThreads), 0, (hipStream_t)stream, a, lanes_log2);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || all) return e;
  const int slices = (a.row_bytes + kSlice - 1) / kSlice;
  hipLaunchKernelGGL(evict_inner_kernel, dim3(heads, (unsigned)(2 * slices + 1 + (a.scales.k ? 2 : 0))),
                     dim3(kMoveThreads), 0, (hipStream_t)stream, a, slices);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  // (no more workgroups than there can be units for)
  const long long most = ((2 * cap << lanes_log2) + 1023) / 1024;
  const long long fill = ((long long)kOuter * kCUs + heads - 1) / heads;
  const unsigned per_head = (unsigned)std::max(1LL, std::min(fill, most));
  hipLaunchKernelGGL(evict_outer_kernel, dim3(heads, per_head), dim3(256), 0, (hipStream_t)stream, a, lanes_log2);
  return hipGetLastError();
}

}  // namespace fa
