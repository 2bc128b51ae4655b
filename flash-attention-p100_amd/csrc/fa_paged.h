// What the kernels over paged caches share: the line of key blocks that deals the
// requests' keys to the waves, a lane's row, and the join of an item's parts. A kernel
// describes itself in T:
//   kD, kBF         the tile's width and the format of q and o (bf16 or fp16)
//   kKeys, kRows    keys of a block, query rows of a tile
//   kTiles, kLine   row tiles that waves abreast take, and the waves that divide a
//                   workgroup's stretch
//   kWaves, kGrid   waves of a workgroup, and workgroups
//   kPUnit          what a weight of 1 counts in the row sums
//   joins()         whether the parts of a workgroup's waves meet before they are written
#pragma once
#include <type_traits>

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

struct PagedKernelArgs {
  const half_t* q;
  half_t* o;
  float* lse;
  const half_t* k;
  const half_t* v;
  long long page_stride, head_stride, row_stride;
  int pages, page_shift;
  const int* table;
  long long table_stride;
  int cap;  // tokens that a table holds
  const int* kv_len;
  float* part_o;    // (wave, 2) x part_rows x D: unscaled partial O
  float2* part_ml;  // (wave, 2) x part_rows: running max (log2 units), row sum
  int4* owned;      // (wave): the item that it begins and does not end (see Owned)
  int* sizes;       // Line's stretch and total
  int part_rows;    // of a tile: kRows, or all of a kv head's
  // items: of a request, groups of row tiles of each kv head
  int B, Hq, group, N, n_groups, items, causal, window, dr;
  bool by_item;  // the kernel's, or the join's, workgroups take an item each
  int runs;  // of 64 or 16 float4 columns in a tile's rows, slice (1 or 2) a join's workgroup
  int slice;
  float scale_log2, rescale, alibi_unit;  // (the last two in units of q . k)
  const float* alibi;
  Strides stq;
};

// A request's keys: [lo, len) are seen by some row, in key blocks first .. first + blocks - 1
// (at least one, so that requests without keys are items too).
template <class T>
struct Keys {
  int len, lo, first, blocks;
  __device__ __forceinline__ Keys(const PagedKernelArgs& a, int raw) {
    len = min(max(raw, 0), a.cap);
    lo = a.window > 0 ? max(0, len - a.N - a.window + 1) : 0;
    first = lo / T::kKeys;
    blocks = max(1, (len + T::kKeys - 1) / T::kKeys - first);
  }
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The sum over the lanes up to each.
__device__ __forceinline__ int wave_prefix(int x) {
  return fa::wave_prefix(x, [](int a, int b) { return a + b; });
}

// The line of key blocks and its division. A request's items are equally long: a
// unit per block and, where every wave has a block or more, `lead` of two before
// them for the item's begin, whose loads nothing runs ahead of. (Of the waves of
// B=250 H=32/4 D=128, up to 600 keys, those with one item took 23 us, with three 30,
// at as many blocks. In all 47 us without the lead, 41 with it; 84 and 64 at B=200
// H=16, up to 400 keys; 22.2 and 21.0 at B=24 H=12 D=64, window 1024.)
template <class T>
struct Line {
  const PagedKernelArgs& a;
  const int lane;
  int lens, c0;      // kv_len of the requests c0 + lane (c0 < 0: none yet)
  int per, through;  // blocks of the requests up to (lane + 1) * per
  int lead;            // units of an item beside its blocks
  int total, stretch;  // all units, and those of a workgroup

  // A line of one item's `units`.
  __device__ __forceinline__ Line(const PagedKernelArgs& a, int lane, int units)
      : a(a), lane(lane), lens(0), c0(0), per(1), through(units), lead(0), total(units), stretch(units) {}
  __device__ __forceinline__ Line(const PagedKernelArgs& a, int lane)
      : a(a), lane(lane), lens(0), c0(a.B > 64 ? -64 : 0), per((a.B + 63) / 64) {
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int c = lane * per + i;
      if (c < a.B) {
        lens = a.kv_len[c];
        mine += Keys<T>(a, lens).blocks * a.items;
      }
    }
    through = wave_prefix(mine);
    total = __builtin_amdgcn_readlane(through, 63);
    stretch = (total + T::kGrid - 1) / T::kGrid;
    lead = stretch >= T::kLine ? 2 : 0;
    if (lead) {
      through += lead * min((lane + 1) * per, a.B) * a.items;
      total += lead * a.B * a.items;
      stretch = (total + T::kGrid - 1) / T::kGrid;
    }
  }
  __device__ __forceinline__ int units(const Keys<T>& k) const { return k.blocks + lead; }
  // The request that holds position pos (< total), and where it starts.
  __device__ __forceinline__ void locate(int pos, int& b, int& start) {
    const int upto = __shfl_up(through, 1), before = lane ? upto : 0;
    const int run = 63 - __clzll(__ballot(before <= pos));
    start = __builtin_amdgcn_readlane(before, run);
    b = run * per;
    if (per == 1) return;
    // (the bounds hold for lengths that another stream changes meanwhile, too)
    for (c0 = b; c0 < a.B; c0 += 64) {
      const int c = c0 + lane;
      lens = a.kv_len[min(c, a.B - 1)];
      const int x = c < min(a.B, (run + 1) * per) ? units(Keys<T>(a, lens)) * a.items : 0;
      const int sum = wave_prefix(x), all = __builtin_amdgcn_readlane(sum, 63);
      if (pos < start + all) {
        const int l = __ffsll(__ballot(start + sum > pos)) - 1;
        b = c0 + l;
        start += __builtin_amdgcn_readlane(sum - x, l);
        return;
      }
      start += all;
    }
    b = a.B - 1;
    start = pos;
  }
  // Where request b starts.
  __device__ __forceinline__ int before(int b) const {
    if (per == 1) return b ? __builtin_amdgcn_readlane(through, b - 1) : 0;
    int sum = 0;
    for (int i = lane; i < b; i += 64) sum += units(Keys<T>(a, a.kv_len[i])) * a.items;
    return __builtin_amdgcn_readlane(wave_prefix(sum), 63);
  }
  __device__ __forceinline__ Keys<T> keys(int b) {
    if ((unsigned)(b - c0) >= 64u) {
      c0 = b;
      lens = a.kv_len[min(b + lane, a.B - 1)];
    }
    return Keys<T>(a, __builtin_amdgcn_readlane(lens, b - c0));
  }
};

// The kernel's arguments, read from memory where this stands. They take about as
// many scalar registers as there are: held from the start, those that the rows and
// results need were spilled ahead of the first loads, 100 instructions that a short
// call waited for (0.8 us at B=8 H=16/4 D=64, 5 tokens).
typedef __attribute__((address_space(4))) const PagedKernelArgs LateArgs;
__device__ __forceinline__ LateArgs& late_args() {
  auto* p = (LateArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// A lane's row of an item's tile of ROWS.
template <int ROWS>
struct Row {
  bool ok;
  int hq, n;
  template <class Args>
  __device__ __forceinline__ Row(const Args& a, int hkv, int tile, int row) {
    const int rows = a.group * a.N, r = tile * ROWS + row, rc = min(r, rows - 1);
    const int g = a.N == 1 ? rc : rc / a.N;
    ok = r < rows;
    hq = hkv * a.group + g;
    n = rc - g * a.N;
  }
};

// Joins the parts of the items that several waves share. A workgroup takes an item
// (by_item), or those that one of paged_kernel's workgroups begins and others end
// (one of each wave at most), and one or two of their runs of 64 float4 columns; its
// waves are dealt to these and then to the parts, so that a long request's parts are
// read in a few rounds. Bound by latency (the lengths, or the list of items that
// paged_kernel left, then the parts: 3.2 to 6 us), so it divides in floats.
constexpr int kMergeWaves = 8;

// x / y for 0 <= x < 2^20, y >= 1: (x + 0.5) / y is 0.5 / y or more from a whole
// number, and off by less than 2^-22 of itself.
__device__ __forceinline__ int small_div(int x, int y) {
  return uniform((int)(((float)x + 0.5f) * __builtin_amdgcn_rcpf((float)y)));
}

// (Six waves per SIMD: up to 80 registers. Left to itself it takes 93, and where the list
// is 1024 workgroups they come in more rounds: 5.0 us against 6.4 at B=60 H=16/2 D=256.)
// RUN: float4 columns of a run. Where they are 16, quarters of a wave take a part each.
template <class T, bool FULL, int RUN>
__global__ __launch_bounds__(64 * kMergeWaves, 6) void paged_merge_kernel(const PagedKernelArgs a) {
  constexpr int D = T::kD, kLine = T::kLine, TILES = T::kTiles, kRows = T::kRows;
  __shared__ floatx4 accs[kMergeWaves][64];
  __shared__ float2 mls[kMergeWaves][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  // (the arguments' four cache lines at once: each takes its time to come)
  asm volatile("" ::"s"(a.o), "s"(a.sizes), "s"(a.part_o), "s"(a.runs), "s"(a.stq.b));
  int stretch, total;
  auto div = [&](int x, int y) { return total < 1 << 17 ? small_div(x, y) : x / y; };
  // The last of a stretch's waves that begins at or before its block x.
  auto wave_of = [&](int x) { return stretch < kLine ? x : div(kLine * (x + 1) - 1, stretch); };
  int4 mine = make_int4(0, 0, 0, 0);
  int g0 = blockIdx.x;
  if (a.by_item) {
    Line<T> line(a, lane);
    const int b = blockIdx.x / a.items;
    int start = line.before(b);
    const int units = line.units(line.keys(b));
    stretch = line.stretch;
    total = line.total;
    const int item = blockIdx.x - b * a.items;
    start += item * units;
    const int last = start + units - 1;
    g0 = div(start, stretch);
    const int owner = wave_of(start - g0 * stretch);
    if (last < (g0 + 1) * stretch &&
        (wave_of(last - g0 * stretch) == owner ||
         (T::joins(stretch, total, a.B * a.items) && start == g0 * stretch &&
          last + 1 == min((g0 + 1) * stretch, total))))
      return;  // (written by its wave or workgroup)
    if (lane == owner) mine = make_int4(b, item, start, units);
  } else {
    stretch = a.sizes[0];
    total = a.sizes[1];
    if (lane < kLine) mine = a.owned[blockIdx.x * kLine + lane];
  }
  const unsigned long long some = __ballot(mine.w > 0);
  if (some == 0) return;
  const int run0 = blockIdx.y * a.slice, runs = min(a.slice, a.runs * TILES - run0);
  const int tasks = __popcll(some) * runs;
  const int per_round = min(tasks, kMergeWaves);
  const int groups = small_div(kMergeWaves, per_round);  // waves that share a task's parts
  const int group = small_div(wave, per_round);
  for (int t0 = 0; t0 < tasks; t0 += kMergeWaves) {
    const int task = t0 + wave - group * per_round;
    bool active = task < tasks && group < groups;
    const int nth = !active ? 0 : TILES == 1 ? task >> (runs - 1) : small_div(task, runs);
    const int part_run = run0 + (active ? task - nth * runs : 0);
    const int beside = TILES == 1 ? 0 : part_run / a.runs, run = part_run - beside * a.runs;
    unsigned long long left = some;
    for (int i = 0; i < nth; ++i) left &= left - 1;
    const int owner = __ffsll(left) - 1;
    const int b = __builtin_amdgcn_readlane(mine.x, owner), item = __builtin_amdgcn_readlane(mine.y, owner);
    const int start = __builtin_amdgcn_readlane(mine.z, owner);
    const int end = start + __builtin_amdgcn_readlane(mine.w, owner);
    // The item's parts: of the waves from `owner` on in its first workgroup (or of
    // the workgroup), of the workgroups between, of the last one's first waves (or
    // of it). Where no stretch is joined, of each block.
    int head = end - start, middle = 0, tail = 0;
    int head_slot = start, first = start, step = 1, middle_slot = 0, tail_slot = 0;
    if (T::joins(stretch, total, a.B * a.items)) {
      const int g1 = div(end - 1, stretch);
      const int x1 = end - g1 * stretch;  // (blocks of the item in g1's stretch, if not all)
      const int last = wave_of(x1 - 1);  // (their last wave)
      const bool whole0 = start == g0 * stretch && g0 < g1, whole1 = end == min((g1 + 1) * stretch, total);
      const int waves = min(kLine, stretch);
      head = whole0 ? 1 : (g0 == g1 ? last + 1 : waves) - owner;
      middle = max(g1 - g0 - 1, 0);
      tail = g0 == g1 ? 0 : whole1 ? 1 : last + 1;
      head_slot = 2 * (g0 * kLine + owner);
      first = head_slot + (whole0 ? 0 : 1);
      step = 2;
      middle_slot = 2 * (g0 + 1) * kLine;
      tail_slot = 2 * g1 * kLine;
    }
    constexpr int kSlots = T::kGrid * kLine * 2;
    const int parts = min(head + middle + tail, kSlots);
    auto slot_of = [&](int p) {
      if (p == 0) return first;
      if (p < head) return head_slot + p * step;
      p -= head;
      return p < middle ? middle_slot + p * 2 * kLine : tail_slot + (p - middle) * 2;
    };
    const int hkv = a.n_groups == 1 ? item : item / a.n_groups;
    const int tile = (item - hkv * a.n_groups) * TILES + beside;
    const int rows = min(kRows, a.group * a.N - tile * kRows);
    active = active && rows > 0;
    constexpr int kSubs = 64 / RUN;
    const int sub = lane / RUN, f = run * RUN + lane % RUN;
    const int rr = min(f / (D / 4), rows - 1), col = 4 * (f % (D / 4));
    float m = -INFINITY, l = 0.f;
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    auto join = [&](float mo, float lo, floatx4 o) {
      const float m_new = fmaxf(m, mo);
      const float keep = m == -INFINITY ? 0.f : fast_exp2(m - m_new);  // (no key: zeros)
      const float add = mo == -INFINITY ? 0.f : fast_exp2(mo - m_new);
      l = l * keep + lo * add;
      acc = acc * keep + o * add;
      m = m_new;
    };
    if (active) {
      const float2* ml = a.part_ml + rr;
      const float* po = a.part_o + rr * D + col;
      constexpr int kAtOnce = 4;
      const int step = groups * kSubs;
      for (int p0 = group * kSubs + sub; p0 < parts; p0 += kAtOnce * step) {
        float2 x[kAtOnce];
        floatx4 o[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (p0 + i * step < parts) {
            const size_t slot =
                (size_t)(min(slot_of(p0 + i * step), kSlots - 1) * TILES + beside) * a.part_rows;
            x[i] = ml[slot];
            o[i] = *reinterpret_cast<const floatx4*>(po + slot * D);
          }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (p0 + i * step < parts) join(x[i].x, x[i].y, o[i]);
      }
#pragma unroll
      for (int x = RUN; x < 64; x <<= 1) {
        const floatx4 o = {__shfl_xor(acc[0], x), __shfl_xor(acc[1], x), __shfl_xor(acc[2], x),
                           __shfl_xor(acc[3], x)};
        join(__shfl_xor(m, x), __shfl_xor(l, x), o);
      }
    }
    // The groups' sums, in halves (0.8 us; one after the other 0.9).
    for (int half = groups >> 1; half > 0; half >>= 1) {
      if (active && group >= half && group < 2 * half) {
        accs[wave][lane] = acc;
        mls[wave][lane] = make_float2(m, l);
      }
      __syncthreads();
      if (active && group < half) {
        const int w = wave + half * per_round;
        join(mls[w][lane].x, mls[w][lane].y, accs[w][lane]);
      }
    }
    if (active && group == 0 && sub == 0 && f < rows * (D / 4)) {
      const Row<kRows> row(a, hkv, tile, rr);
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (FULL || col < a.dr) {
        half4 o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = to16<T::kBF>(acc[e] * inv);
        *reinterpret_cast<half4*>(a.o + b * a.stq.b + row.hq * a.stq.h + (size_t)row.n * a.stq.n + col) = o4;
      }
      if (col == 0 && a.lse)
        a.lse[((size_t)b * a.Hq + row.hq) * a.N + row.n] =
            l == 0.f ? INFINITY : (m + __log2f(l * T::kPUnit)) * kLn2;
    }
  }
}

// The workspace: two parts of each wave (unscaled O, maximum and sum of its rows), the
// list of the items that waves begin, the line's sizes.
template <class T>
size_t paged_workspace(int rows) {
  constexpr size_t kAll = (size_t)T::kGrid * T::kWaves;
  return kAll * 2 * min(rows, T::kRows) * (T::kD * sizeof(float) + sizeof(float2)) +
         kAll * sizeof(int4) + 2 * sizeof(int);
}

template <class T>
void paged_args(PagedKernelArgs& d, const PagedArgs& a) {
  d.q = (const half_t*)a.q;
  d.o = (half_t*)a.o;
  d.lse = a.lse;
  d.k = (const half_t*)a.pool.k;
  d.v = (const half_t*)a.pool.v;
  d.page_stride = a.pool.page_stride;
  d.head_stride = a.pool.head_stride;
  d.row_stride = a.pool.row_stride;
  d.pages = a.pool.pages;
  d.page_shift = a.pool.page_shift;
  d.table = a.table;
  d.table_stride = a.table_stride;
  d.cap = a.table_width << a.pool.page_shift;
  d.kv_len = a.kv_len;
  d.B = a.B;
  d.Hq = a.Hq;
  d.group = a.Hq / a.Hkv;
  d.N = a.N;
  d.part_rows = min(d.group * a.N, T::kRows);
  d.part_o = (float*)a.workspace;
  constexpr size_t kAll = (size_t)T::kGrid * T::kWaves;
  d.part_ml = (float2*)(d.part_o + kAll * 2 * d.part_rows * T::kD);
  d.owned = (int4*)(d.part_ml + kAll * 2 * d.part_rows);
  d.sizes = (int*)(d.owned + kAll);
  const int n_tiles = (d.group * a.N + T::kRows - 1) / T::kRows;
  d.n_groups = (n_tiles + T::kTiles - 1) / T::kTiles;
  d.items = a.Hkv * d.n_groups;
  d.causal = a.causal;
  d.window = a.window < d.cap ? a.window : 0;  // (a wider one hides nothing)
  d.dr = a.D;
  d.scale_log2 = kLog2e * (a.scale > 0.f ? a.scale : 1.f / sqrtf((float)a.D));
  d.rescale = T::kPRescale / d.scale_log2;
  d.alibi_unit = kLog2e / d.scale_log2;
  d.alibi = a.alibi;
  d.stq = make_strides(a.layout, a.Hq, a.N, a.D);
}

template <class T, bool FULL>
hipError_t launch_paged_join(PagedKernelArgs& d, hipStream_t stream) {
  // A join workgroup per item and run where these are at most half as many as the
  // list's (3.8 us against 4.8 at B=8 H=16/4 D=64, 5 tokens: 160 and 768 workgroups;
  // 4.6 against 6.1 at B=30 H=16/2 D=256: 480 and 1024); else the list, a shorter way to
  // the parts (4.3 against 7.8 at B=40 H=16/4 D=64, 4 tokens: 512 and 640; 6.5 against
  // 13.4 at B=100 H=16/2 D=256: 1024 and 1600), with two runs each (1.3 us less
  // than with one at B=250 H=32/4 D=128). The list too for items of one run, but for
  // up to four of them, whose parts can be many (at B=1 H=16/4 D=64: 4.2 us against
  // 4.9 at 4000 keys, 3.9 and 3.4 at 1000).
  const long long items = (long long)d.B * d.items;
  const int columns = d.part_rows * (T::kD / 4);
  d.runs = (columns + 63) / 64;
  d.by_item = (d.runs > 1 || items <= 4) &&
              2 * items * d.runs * T::kTiles <= T::kGrid * ((d.runs * T::kTiles + 1) / 2);
  // Of 16 columns where few workgroups would join many parts: 5.8 us for 9.0 at B=1 H=8/1
  // D=128, 20000 keys (4 workgroups, 16 with shorter runs).
  const bool narrow = d.by_item && items * d.runs * T::kTiles <= 64;
  if (narrow) d.runs = (columns + 15) / 16;
  d.slice = d.by_item ? 1 : 2 * T::kTiles;
  const unsigned slices = (unsigned)((d.runs * T::kTiles + d.slice - 1) / d.slice);
  const auto merge = narrow ? paged_merge_kernel<T, FULL, 16> : paged_merge_kernel<T, FULL, 64>;
  hipLaunchKernelGGL(merge, dim3(d.by_item ? (unsigned)items : T::kGrid, slices),
                     dim3(64 * kMergeWaves), 0, stream, d);
  return hipGetLastError();
}

}  // namespace
}  // namespace fa
