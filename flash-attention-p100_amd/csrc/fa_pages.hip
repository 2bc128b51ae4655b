// Paged key/value caches: the block tables and slots of a step from the
// requests' lengths, and the writes of new rows into their slots. No counterpart
// in the reference, which has no cache. (The attention over them: fa_paged.hip.)
#include <algorithm>

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

}  // namespace

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
