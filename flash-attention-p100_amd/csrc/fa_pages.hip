// Paged key/value caches: the block tables and slots of a step from the
// requests' lengths, the writes of new rows into their slots, in 16 bits or
// quantised to 4, and rows read back from there. No counterpart in the reference,
// which has no cache. (The attention over them: fa_paged.hip, fa_paged4.hip.)
#include <algorithm>
#include <type_traits>

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

// ---------------------------------------------------------------------------
// Tables and slots. With p rows per page, request b of old and new lengths o, n
// owns ceil(o / p) pages and wants ceil(n / p): the pages it takes are the free
// ring's entries from head + (what the requests before it take) on, those it
// gives back go behind the ring's last free entry likewise. Everything follows
// from three prefix sums over the requests (pages taken, pages returned, tokens
// added), which every workgroup computes for itself, a tile of requests at a
// time: the lengths are a few KB in L2, and a launch apart for the sums would
// cost more than the call. The workgroups then share the tile's pages and
// tokens evenly, finding a page's or token's request by bisection in LDS, so one
// long prompt is spread like many short ones. Nothing that a workgroup reads is
// written in the launch: taken pages come from the ring (a token's slot looks
// there too, not into the table), returned ones from table entries that no
// taken page replaces, and the free entries they overwrite are none of the
// ring's. Bound by latency: the lengths, a bisection, the page.
constexpr int kTabThreads = 256;  // and requests per tile

// Sums saturate at 2^31 - 1, which is past every ring, table and slot array.
__device__ __forceinline__ int sat_add(int a, int b) {
  return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu);
}
struct Sums {
  int need, gone, grown;  // pages to take and to return, tokens added
};
__device__ __forceinline__ Sums operator+(Sums a, Sums b) {
  return {sat_add(a.need, b.need), sat_add(a.gone, b.gone), sat_add(a.grown, b.grown)};
}

struct Request {
  int old, have, want, capped, grown;  // tokens and pages before, pages and tokens wanted, new ones
  __device__ __forceinline__ Request(const TablesArgs& a, int b)
      : old(0), have(0), want(0), capped(0), grown(0) {
    if (b >= a.B) return;
    const int cap = a.table_width << a.page_shift, n = max(a.new_len[b], 0);
    old = min(max(a.old_len[b], 0), cap);
    capped = min(n, cap);
    have = pages(a, old);
    want = pages(a, capped);
    grown = max(n - old, 0);
  }
  __device__ __forceinline__ static int pages(const TablesArgs& a, int len) {
    return (int)(((unsigned)len + (1u << a.page_shift) - 1u) >> a.page_shift);
  }
};

// The first of `n` ascending values that is greater than x (n if none is).
__device__ __forceinline__ int first_above(const int* v, int n, int x) {
  int lo = 0;
  for (int hi = n; lo < hi;) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// PER: slots in a row that a thread finds.
template <int PER>
__global__ __launch_bounds__(kTabThreads) void tables_kernel(const TablesArgs a) {
  // Of the tile's requests: the sums through each, and what a token needs.
  __shared__ int need_end[kTabThreads], gone_end[kTabThreads], grown_end[kTabThreads];
  __shared__ int olds[kTabThreads], haves[kTabThreads], wants[kTabThreads], lens[kTabThreads];
  __shared__ Sums waves[kTabThreads / 64];
  const int tid = threadIdx.x, C = a.n_ring;
  const int behind = a.ring[0] % C, head = behind < 0 ? behind + C : behind;
  const int count = min(max(a.ring[1], 0), C);
  const int page_mask = (1 << a.page_shift) - 1;
  const bool packed = a.tokens >= 0;
  Sums carry{0, 0, 0};  // of the tiles before
  // The ring's entry i (below C) past the head.
  auto ring_at = [&](int i) { return head + i < C ? head + i : head + i - C; };
  // Where request r's (of the tile) page p stands: its own, or one that it takes now.
  auto entry_of = [&](int b, int r, int p) -> const int* {
    const int before = r ? need_end[r - 1] : carry.need;
    return p < haves[r] ? a.table + b * a.table_stride + p : a.free_pages + ring_at(before + p - haves[r]);
  };
  const bool vec = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  for (int b0 = 0; b0 < a.B; b0 += kTabThreads) {
    const int b = b0 + tid;
    const Request q(a, b);
    Sums s{max(q.want - q.have, 0), max(q.have - q.want, 0), q.grown};
    s = {wave_prefix(s.need, sat_add), wave_prefix(s.gone, sat_add), wave_prefix(s.grown, sat_add)};
    if ((tid & 63) == 63) waves[tid >> 6] = s;
    __syncthreads();
    s = s + carry;
    for (int w = 0; w < (tid >> 6); ++w) s = s + waves[w];
    need_end[tid] = s.need;
    gone_end[tid] = s.gone;
    grown_end[tid] = s.grown;
    olds[tid] = q.old;
    haves[tid] = q.have;
    wants[tid] = q.want;
    const int need = max(q.want - q.have, 0);
    // (past saturation nothing is left to give)
    const int given = min(need, max(count - (s.need - need), 0));
    const int held = (q.have + given) << a.page_shift;  // (at most the table's tokens)
    lens[tid] = q.capped > q.old ? min(q.capped, held) : q.capped;
    if (b < a.B && blockIdx.x == 0) a.kv_len[b] = lens[tid];
    __syncthreads();
    const int n = min(kTabThreads, a.B - b0);
    // The tile's pages taken (up to the free ones), pages returned (as far as the
    // ring has room) and groups of PER slots, one run of items for all workgroups.
    const int takes = max(min(need_end[n - 1], count) - carry.need, 0);
    const int returns = max(min(gone_end[n - 1], C - count) - carry.gone, 0);
    const int s0 = packed ? min(carry.grown, a.tokens) : b0 * a.max_new;
    const int s1 = packed ? min(grown_end[n - 1], a.tokens) : (b0 + n) * a.max_new;
    const long long groups = s1 > s0 ? (s1 - 1) / PER - s0 / PER + 1 : 0;
    const long long items = takes + returns + groups;
    for (long long i = (long long)blockIdx.x * kTabThreads + tid; i < items;
         i += (long long)gridDim.x * kTabThreads) {
      if (i < takes) {
        const int x = carry.need + (int)i, r = first_above(need_end, n, x);
        const int p = haves[r] + x - (r ? need_end[r - 1] : carry.need);
        a.table[(b0 + r) * a.table_stride + p] = a.free_pages[ring_at(x)];
      } else if (i < takes + (long long)returns) {
        const int x = carry.gone + (int)(i - takes), r = first_above(gone_end, n, x);
        const int p = wants[r] + x - (r ? gone_end[r - 1] : carry.gone);
        a.free_pages[ring_at(count + x)] = a.table[(b0 + r) * a.table_stride + p];
      } else {
        // Slots g .. g + PER - 1, as far as they are the tile's. (g + e stays below 2^31: s1 does.)
        const int g = (s0 / PER + (int)(i - takes - returns)) * PER;
        const int from = max(g, s0), upto = (int)min((long long)g + PER, (long long)s1);
        int r, first;  // the request of slot `from`, and the slot of its first new token
        if (packed) {
          r = first_above(grown_end, n, from);
          first = r ? grown_end[r - 1] : carry.grown;
        } else {
          r = a.max_new == 1 ? from - s0 : (from - s0) / a.max_new;
          first = s0 + r * a.max_new;
        }
        // (the loads at once; where there is no token, of the ring's head)
        const int* entry[PER];
        int row[PER], slots[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int x = g + e;
          entry[e] = a.ring;
          row[e] = -1;
          if (x < from || x >= upto) continue;
          while (x >= (packed ? grown_end[r] : first + a.max_new)) {
            first = packed ? grown_end[r] : first + a.max_new;
            ++r;
          }
          const unsigned j = (unsigned)olds[r] + (unsigned)(x - first);
          if (j >= (unsigned)lens[r]) continue;
          entry[e] = entry_of(b0 + r, r, (int)(j >> a.page_shift));
          row[e] = (int)j & page_mask;
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) slots[e] = *entry[e];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const long long slot = ((long long)slots[e] << a.page_shift) + row[e];
          slots[e] = row[e] < 0 || slots[e] < 0 || slot > 0x7fffffffLL ? -1 : (int)slot;
        }
        if (PER == 4 && vec && from == g && upto == g + PER) {
          *reinterpret_cast<int4*>(a.slots + g) = make_int4(slots[0], slots[1 % PER], slots[2 % PER], slots[3 % PER]);
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (g + e >= from && g + e < upto) a.slots[g + e] = slots[e];
        }
      }
    }
    carry = {need_end[n - 1], gone_end[n - 1], grown_end[n - 1]};
    __syncthreads();
  }
  if (packed)  // behind the last token
    for (long long i = (long long)carry.grown + blockIdx.x * kTabThreads + tid; i < a.tokens;
         i += (long long)gridDim.x * kTabThreads)
      a.slots[i] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    const int taken = min(carry.need, count);
    a.ring_out[0] = taken < C ? ring_at(taken) : head;
    a.ring_out[1] = count - taken + min(carry.gone, C - count);
  }
}

// ---------------------------------------------------------------------------
// Cache writes: a copy of each token's K and V rows to its slot, a thread per
// 16-byte chunk, workgroups of K and of V in turn (both in one thread: 96 us where
// this takes 88, into pages that hold the rows before the heads). Bound by HBM at
// prompts (88 to 92 us for 65536 tokens of 8 heads of 128, 529 MB moved at 5.8 TB/s
// or more; a copy of 2 GiB moves 4.95), by latency at a step (2.7 us for 64 tokens).
constexpr int kAppThreads = 256;
// Chunks from which loads and stores carry the nontemporal hint: 32 MB written, what
// the L2s hold. Above, the hint takes 98 to 88 us at 268 MB and 27.4 to 24.3 at 67;
// below, rows that L2 would have taken wait for memory (6.5 us without it and 8.0
// with it at 17 MB).
constexpr long long kAppStream = 1LL << 20;

struct AppendArgs {
  const half_t* from[2];  // k and v, their strides and their pools
  RowStrides strides[2];
  half_t* to[2];
  const int* slots;
  long long page_stride, head_stride, row_stride;
  int pages, page_shift;
  int N, row_chunks, chunks;  // 16-byte chunks of a row, and of a token's heads
  long long items;            // tokens * chunks
};

template <class Index, bool STREAM>  // (division of 64 bits takes longer than a step's copy)
__global__ __launch_bounds__(kAppThreads) void append_kernel(const AppendArgs a) {
  const bool v = blockIdx.x & 1;
  const half_t* const from = v ? a.from[1] : a.from[0];
  const RowStrides s = v ? a.strides[1] : a.strides[0];
  half_t* const to = v ? a.to[1] : a.to[0];
  const Index step = (Index)(gridDim.x / 2) * kAppThreads, items = (Index)a.items;
  for (Index i = (Index)(blockIdx.x / 2) * kAppThreads + threadIdx.x; i < items; i += step) {
    const int t = (int)(i / (Index)a.chunks), x = (int)(i - (Index)t * a.chunks);
    const int slot = a.slots[t], page = slot >> a.page_shift;
    if (slot < 0 || page >= a.pages) continue;
    const int h = x / a.row_chunks, c = (x - h * a.row_chunks) * 8;
    const int b = a.N == 1 ? t : t / a.N, n = t - b * a.N;
    const u32x4* src = reinterpret_cast<const u32x4*>(from + b * s.b + n * s.n + h * s.h + c);
    u32x4* dst = reinterpret_cast<u32x4*>(to + page * a.page_stride + h * a.head_stride +
                                          (slot - (page << a.page_shift)) * a.row_stride + c);
    if constexpr (STREAM) __builtin_nontemporal_store(__builtin_nontemporal_load(src), dst);
    else *dst = *src;
  }
}

// ---------------------------------------------------------------------------
// Writes into a cache in 4 bits. With m the largest magnitude of 32 values of a row,
// their scale is the least power of two X (from 2^-126 on) with m <= 7 X, so m keeps a
// code next to it (up to 8 X, as the usual choice allows, the largest would be clamped
// from 8 to 6), and a value x becomes the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to
// |x| / X, ties to the even code, with x's sign. x / X is exact, so the codes are those
// that any correct rounding gives. Four lanes hold a block, a 16-byte chunk each.
template <bool BF>
__device__ __forceinline__ uint32_t to_codes(u32x4 x, float scale) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  uint32_t c = 0;
  auto two = [&](uint32_t pair, auto sel) {
    constexpr int kByte = decltype(sel)::value;
    if constexpr (BF) c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf2, pair), scale, kByte);
    else c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(half2, pair), scale, kByte);
  };
  two(x[0], std::integral_constant<int, 0>{});
  two(x[1], std::integral_constant<int, 1>{});
  two(x[2], std::integral_constant<int, 2>{});
  two(x[3], std::integral_constant<int, 3>{});
  return c;
}

// The largest scales, of which 6 times is finite in the rows' format.
template <bool BF>
constexpr uint32_t kTopScale = BF ? 127 + 125 : 127 + 13;

struct RowsArgs {
  const half_t* from[2];  // dense rows: k and v, their strides
  half_t* into[2];
  RowStrides strides[2];
  uint8_t* codes[2];  // the pools, and their scales (16-bit rows: none)
  uint8_t* scales[2];
  const int* slots;
  uint32_t page_stride, row_stride, scale_page, scale_row;  // in bytes
  long long head_stride, scale_head;
  int pages, page_shift;
  uint32_t tokens;
  int N, row_chunks, chunks;  // 16-byte chunks of a dense row, and of a token's heads
  int width, per;             // chunks of a token, and tokens, that a workgroup takes at once
  int step, step_n;           // a thread's next token, and by how many rows in its request
  long long hop[2], hop_next[2];  // as far in the dense rows: within a request, to the next
};

// The chunk of a token that a thread moves.
struct Chunk {
  int v, h, c;
};
// A token's place in the pools, or none: page < 0.
struct Place {
  int page, row;
  __device__ __forceinline__ Place() {}
  __device__ __forceinline__ Place(const RowsArgs& a, uint32_t t) {
    const int slot = a.slots[min(t, a.tokens - 1)];
    page = slot >> a.page_shift;
    row = slot - (page << a.page_shift);
    if (t >= a.tokens || page >= a.pages) page = -1;
  }
  __device__ __forceinline__ uint64_t in_pool(const RowsArgs& a) const {
    return (uint64_t)(uint32_t)page * a.page_stride + (uint64_t)(uint32_t)row * a.row_stride;
  }
  __device__ __forceinline__ uint64_t in_scales(const RowsArgs& a) const {
    return (uint64_t)(uint32_t)page * a.scale_page + (uint64_t)(uint32_t)row * a.scale_row;
  }
};

// Goes over the chunks: a thread keeps its place within the tokens and goes from token to
// token, COUNT at a time, so that it divides once. load(chunk, place, dense offset) for all
// of them (any token's where theirs is missing), then done(chunk, place, dense offset, what
// was loaded). Both directions are bound by HBM: 65536 tokens of 8 heads of 128 are written
// in 65 us and read back in 56 (340 MB each), with a chunk to a thread, found by division
// (150 instructions each, and bound by them), 94 each, and without the streaming hint for
// the dense rows 77 and 70.
template <int COUNT, class Load, class Done>
__device__ __forceinline__ void each_chunk(const RowsArgs& a, Load&& load, Done&& done) {
  const int v = blockIdx.x & 1, sub = threadIdx.x / a.width;
  const int x = blockIdx.y * kAppThreads + (int)threadIdx.x - sub * a.width;
  if (sub >= a.per || x >= a.chunks) return;
  const int h = x / a.row_chunks;
  const Chunk chunk{v, h, x - h * a.row_chunks};
  const RowStrides s = v ? a.strides[1] : a.strides[0];
  const long long hop = v ? a.hop[1] : a.hop[0], hop_next = v ? a.hop_next[1] : a.hop_next[0];
  uint32_t t = (blockIdx.x >> 1) * a.per + sub;
  if (t >= a.tokens) return;
  const int b = t / a.N;
  const uint32_t N = (uint32_t)a.N;
  uint32_t n = t - (uint32_t)b * N;
  long long at = b * s.b + n * s.n + h * s.h + 8 * chunk.c;
  for (; t < a.tokens; t += COUNT * a.step) {
    Place places[COUNT];
    long long dense[COUNT];
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      places[e] = Place(a, t + e * a.step);
      dense[e] = t + e * a.step < a.tokens ? at : dense[0];
      n += a.step_n;
      at += n >= N ? hop_next : hop;
      n -= n >= N ? N : 0;
    }
    decltype(load(chunk, places[0], at)) x[COUNT];
#pragma unroll
    for (int e = 0; e < COUNT; ++e) x[e] = load(chunk, places[e], dense[e]);
#pragma unroll
    for (int e = 0; e < COUNT; ++e)
      if (t + e * a.step < a.tokens) done(chunk, places[e], dense[e], x[e]);
  }
}

template <bool BF, int COUNT>
__global__ __launch_bounds__(kAppThreads) void append4_kernel(const RowsArgs a) {
  const half_t* const from = blockIdx.x & 1 ? a.from[1] : a.from[0];
  uint8_t* const codes = blockIdx.x & 1 ? a.codes[1] : a.codes[0];
  uint8_t* const scales = blockIdx.x & 1 ? a.scales[1] : a.scales[0];
  auto load = [&](const Chunk&, const Place&, long long dense) {
    const u32x4* const at = reinterpret_cast<const u32x4*>(from + dense);
    return COUNT > 1 ? __builtin_nontemporal_load(at) : *at;
  };
  auto done = [&](const Chunk& x, const Place& at, long long, u32x4 in) {
    if (at.page < 0) return;  // (all four lanes of a block: one row)
    // (magnitudes of 16 bits are in the order of their bits)
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, in[e] & 0x7fff7fffu));
    int top = max((int)m[0], (int)m[1]);
    top = max(top, __builtin_amdgcn_update_dpp(0, top, 0xb1, 0xf, 0xf, false));  // lane ^ 1
    top = max(top, __builtin_amdgcn_update_dpp(0, top, 0x4e, 0xf, 0xf, false));  // lane ^ 2
    const half_t top16 = __builtin_bit_cast(half_t, (unsigned short)top);
    const uint32_t bits = __float_as_uint(from16<BF>(top16));
    // (one more above 1.75 of its power of two)
    uint32_t e = (uint32_t)min(max((int)((bits + 0x1fffffu) >> 23) - 2, 1), (int)kTopScale<BF>);
    uint32_t out = to_codes<BF>(in, __uint_as_float(e << 23));
    if (bits >= 0x7f800000u) {  // an infinity or a NaN: the block is NaN
      e = 255;
      out = 0;
    }
    *reinterpret_cast<uint32_t*>(codes + at.in_pool(a) + x.h * a.head_stride + 4 * x.c) = out;
    if ((x.c & 3) == 0) scales[at.in_scales(a) + x.h * a.scale_head + (x.c >> 2)] = (uint8_t)e;
  };
  each_chunk<COUNT>(a, load, done);
}

// ---------------------------------------------------------------------------
// Rows back from their slots, dense: 16-bit ones as they are, 4-bit ones as the values
// that they stand for, exact in bf16 and rounded to nearest even in fp16. Rows without a
// slot are zeros. FOUR: the cache is in 4 bits.
template <bool BF, bool FOUR, int COUNT>
__global__ __launch_bounds__(kAppThreads) void gather_kernel(const RowsArgs a) {
  half_t* const into = blockIdx.x & 1 ? a.into[1] : a.into[0];
  const uint8_t* const codes = blockIdx.x & 1 ? a.codes[1] : a.codes[0];
  const uint8_t* const scales = blockIdx.x & 1 ? a.scales[1] : a.scales[0];
  struct Cached {
    u32x4 x;
    uint32_t scale;
  };
  auto load = [&](const Chunk& x, Place at, long long) {
    if (at.page < 0) at.page = at.row = 0;
    const uint8_t* const row = codes + at.in_pool(a) + x.h * a.head_stride;
    if constexpr (FOUR)
      return Cached{{*reinterpret_cast<const uint32_t*>(row + 4 * x.c), 0u, 0u, 0u},
                    scales[at.in_scales(a) + x.h * a.scale_head + (x.c >> 2)]};
    else
      return Cached{*reinterpret_cast<const u32x4*>(row + 16 * x.c), 0u};
  };
  auto done = [&](const Chunk&, const Place& at, long long dense, const Cached& in) {
    u32x4 out = in.x;
    if constexpr (FOUR) {
      const uint32_t x = in.x[0];
      const float scale = __uint_as_float(in.scale << 23);
      auto two = [&](auto sel) {
        if constexpr (BF)
          return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, decltype(sel)::value));
        const auto f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, decltype(sel)::value);
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(_Float16)f[0], (_Float16)f[1]});
      };
      out = u32x4{two(std::integral_constant<int, 0>{}), two(std::integral_constant<int, 1>{}),
                  two(std::integral_constant<int, 2>{}), two(std::integral_constant<int, 3>{})};
    }
    if (at.page < 0) out = u32x4{0u, 0u, 0u, 0u};
    u32x4* const to = reinterpret_cast<u32x4*>(into + dense);
    if constexpr (COUNT > 1)
      __builtin_nontemporal_store(out, to);
    else
      *to = out;
  };
  each_chunk<COUNT>(a, load, done);
}

RowsArgs rows_args(RowStrides sk, RowStrides sv, const int* slots, const PagedPool& pool,
                   const PagedScales* scales, int B, int N, int Hkv, int D) {
  RowsArgs a{};
  a.strides[0] = sk;
  a.strides[1] = sv;
  a.codes[0] = (uint8_t*)pool.k;
  a.codes[1] = (uint8_t*)pool.v;
  const int unit = scales ? 1 : 2;  // (16-bit pools' strides count elements)
  a.page_stride = (uint32_t)(unit * pool.page_stride);
  a.head_stride = unit * pool.head_stride;
  a.row_stride = (uint32_t)(unit * pool.row_stride);
  if (scales) {
    a.scales[0] = scales->k;
    a.scales[1] = scales->v;
    a.scale_page = (uint32_t)scales->page_stride;
    a.scale_head = scales->head_stride;
    a.scale_row = (uint32_t)scales->row_stride;
  }
  a.slots = slots;
  a.pages = pool.pages;
  a.page_shift = pool.page_shift;
  a.tokens = (uint32_t)B * N;
  a.N = N;
  a.row_chunks = D / 8;
  a.chunks = Hkv * a.row_chunks;
  a.width = std::min(a.chunks, kAppThreads);
  a.per = kAppThreads / a.width;
  return a;
}

// Launches kernel_of(COUNT): several chunks to a thread where the card is full (kRowsPerCu
// workgroups to a CU; with 8 the calls above take 67 and 59 us, with 64 74 and 53).
constexpr int kRowsPerCu = 16;
template <class KernelOf>
hipError_t launch_rows(RowsArgs& a, const KernelOf& kernel_of, void* stream) {
  const unsigned slices = (unsigned)((a.chunks + kAppThreads - 1) / kAppThreads);
  const unsigned all = (a.tokens + a.per - 1) / a.per;
  const unsigned most = std::max(1u, (unsigned)(kRowsPerCu * kCUs) / (2 * slices));
  const unsigned blocks = std::min(all, most);
  a.step = (int)blocks * a.per;
  const long long step_b = a.step / a.N;
  a.step_n = a.step % a.N;
  for (int v = 0; v < 2; ++v) {
    a.hop[v] = step_b * a.strides[v].b + a.step_n * a.strides[v].n;
    a.hop_next[v] = a.hop[v] + a.strides[v].b - a.N * a.strides[v].n;
  }
  const auto kernel = all > most ? kernel_of(std::integral_constant<int, 4>{})
                                 : kernel_of(std::integral_constant<int, 1>{});
  hipLaunchKernelGGL(kernel, dim3(2 * blocks, slices), dim3(kAppThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged4_append(const void* k, const void* v, RowStrides sk, RowStrides sv,
                                const int* slots, const PagedPool& pool, const PagedScales& scales,
                                int B, int N, int Hkv, int D, int dtype, void* stream) {
  RowsArgs a = rows_args(sk, sv, slots, pool, &scales, B, N, Hkv, D);
  a.from[0] = (const half_t*)k;
  a.from[1] = (const half_t*)v;
  return launch_rows(
      a, [&](auto n) { return dtype == kBF16 ? append4_kernel<true, n()> : append4_kernel<false, n()>; }, stream);
}

hipError_t launch_paged_gather(void* k, void* v, RowStrides strides, const int* slots,
                               const PagedPool& pool, const PagedScales* scales, int B, int N,
                               int Hkv, int D, int dtype, void* stream) {
  RowsArgs a = rows_args(strides, strides, slots, pool, scales, B, N, Hkv, D);
  a.into[0] = (half_t*)k;
  a.into[1] = (half_t*)v;
  return launch_rows(
      a,
      [&](auto n) {
        return !scales          ? gather_kernel<true, false, n()>
               : dtype == kBF16 ? gather_kernel<true, true, n()>
                                : gather_kernel<false, true, n()>;
      },
      stream);
}

hipError_t launch_paged_tables(const TablesArgs& a, void* stream) {
  // Four slots per thread from 32768 on (6.2 us for 350000 packed ones, 7.9 one at a
  // time), one below (3.3 us for a step of 64 requests, 4.3 with four). The requests'
  // sums are done again in each workgroup, so these are at most two per CU.
  const long long slots = a.tokens >= 0 ? a.tokens : (long long)a.B * a.max_new;
  const int per = slots >= 32768 ? 4 : 1;
  const unsigned blocks =
      (unsigned)std::min((std::max(slots, 1LL) + kTabThreads * per - 1) / (kTabThreads * per), 512LL);
  if (per == 4)
    hipLaunchKernelGGL(tables_kernel<4>, dim3(blocks), dim3(kTabThreads), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(tables_kernel<1>, dim3(blocks), dim3(kTabThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_append(const void* k, const void* v, RowStrides sk, RowStrides sv,
                               const int* slots, const PagedPool& pool, int B, int N, int Hkv,
                               int D, void* stream) {
  AppendArgs a{{(const half_t*)k, (const half_t*)v}, {sk, sv}, {(half_t*)pool.k, (half_t*)pool.v}, slots};
  a.page_stride = pool.page_stride;
  a.head_stride = pool.head_stride;
  a.row_stride = pool.row_stride;
  a.pages = pool.pages;
  a.page_shift = pool.page_shift;
  a.N = N;
  a.row_chunks = D / 8;
  a.chunks = Hkv * a.row_chunks;
  a.items = (long long)B * N * a.chunks;
  const unsigned blocks = 2 * (unsigned)std::min((a.items + kAppThreads - 1) / kAppThreads, 1LL << 20);
  // (32 bits while i + step stays below 2^32)
  const auto kernel = a.items < kAppStream    ? append_kernel<uint32_t, false>
                      : a.items <= 1LL << 31 ? append_kernel<uint32_t, true>
                                             : append_kernel<uint64_t, true>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kAppThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError();
}

}  // namespace fa
