// Attention of the newest tokens of each request over its paged key/value cache
// (tables and cache writes: fa_pages.hip). No counterpart in the reference,
// which has no cache.
//
// Bound: HBM, each K/V row is read once per 32 to 128 query rows. As in fa_dec.hip a row
// tile is 32 rows of one kv head (the rows of the query heads of its group, head
// after head), a wave's step is a block of 32 keys of its own LDS tiles, and the
// products are S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16. What is
// different is where the keys are and how they are dealt out:
//   * the lengths are known on the device only, and differ. So all key blocks of
//     the call, request after request, kv head after kv head, tile after tile, lie
//     on one line, which the waves divide evenly: each finds its stretch from the
//     sum of the lengths, walks the items (a row tile of a request's kv head) in
//     it, and writes the result of an item that it has whole; the parts of the
//     others meet in paged_merge_kernel. No wave waits for a longer request. Where
//     a workgroup's stretch lies within one item, its waves' parts meet in LDS
//     first: long requests then leave one where the kLine waves that divide the
//     stretch (8, 4 at D=256, less with tiles abreast) would leave one each. Several
//     row tiles of a kv head go side by side, as many waves over the same stretch;
//   * a wave's lanes hold the next 64 page indices of its stretch; a block's rows
//     take theirs from there by a lane permutation, so the table is read once in
//     64 pages and the K/V loads (direct to LDS, an address per lane) wait for
//     nothing. Rows outside the request's keys read one of its rows instead: a
//     masked key's P is zero, but zero times what an unused row holds may be NaN.
// Measured at D=128, bf16: 399 us and 7 for the join at B=64 H=32/8, up to 16384
// keys (2.6 GB, 6.5 TB/s; the fastest large read found reaches 7.1, most others 6);
// 6.6 and 3.8 us for one request of 1021 keys, H=16/8, most of it the way to the first
// keys and to the parts.
#include <type_traits>

#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

constexpr int kRows = 32;  // query rows of a tile
constexpr int kKeys = 32;  // keys of a wave's block

// P = 2^(kPScale + log2 units of a score below its row's maximum) is rounded to the
// inputs' format as the second product's operand. Up to 32 rows per kv head a second
// matrix instruction adds the product of what that rounding left, itself rounded (P is
// off by 2^-16 of itself in bf16 and 2^-22 in fp16), so the results are off the 64-bit
// ones by their own rounding (0.0017 of their norm in bf16, 0.00021 in fp16; 0.0020 to
// 0.0023 and 0.00024 to 0.00027 without). HBM bounds these calls: 0.2 to 0.5 us of 10
// to 40, 1 of 160, none of 400. With more rows the instructions bound, and P is rounded
// once, as in the other forward kernels (another product would take 113 us to 115 at
// B=20 H=64/8 D=128, 8 tokens, and 51 to 57 at D=64; 146 to 157 at 16 tokens; 490 to 580
// for 2048 tokens of H=32/8 D=128 over 8192).
//
// bf16 has fp32's exponents. fp16's end at 2^-24, which the many small weights behind
// one large one (an attention sink) may be below, so P is 2^15 there for the row's
// largest and the maximum is never behind: half a step holds down to 2^-29 of the
// largest, and 2^-40 of it below. (With P up to 2^8 and none of the scale, as in the
// other forward kernels, a tail of 16384 keys at 2^-24.5 came out 1.5 times too large.)
// Each time that a row's maximum grows O is multiplied; where the products bound, that
// took 1 to 3% (140 us for 138 and 503 for 487 at 512 and 2048 tokens of H=32/8 D=128
// over 8192).
template <bool BF>
constexpr int kPScale = BF ? 0 : 15;
template <bool BF>
constexpr float kPUnit = BF ? 1.f : 0x1p-15f;
// The maximum's growth, in log2 units, that leaves it where it was.
template <bool BF>
constexpr float kPRescale = BF ? kRescaleLog2 : 0.f;

template <int D>
struct Paged {
  static constexpr int kWaves = D > 128 ? 4 : 8;
  static constexpr int kThreads = 64 * kWaves;
  // Row tiles of a kv head that waves abreast take, over the same keys, and the waves
  // of each: what one brings in the others find in L2. (In all 113 us for 146 at B=20
  // H=64/8 D=128, 7 tokens, up to 8000 keys, and 208 for 296 at D=256; tiles apart on
  // the line read from HBM each, and are better where L2 holds all: 14.1 for 14.6 at
  // B=1 H=64/8 D=128, 5 tokens, 2000 keys.)
  template <int TILES>
  static constexpr int kLine = kWaves / TILES;
  // Waves per SIMD that the compiler is to allow for. More than run, but asked for less
  // it spills scalar registers, 33 instead of 3 at D=64 (15.6 us in all for 15.2 at
  // B=60 H=16/4, up to 1000 keys).
  static constexpr int kPerSimd = D == 32 ? 4 : D == 64 ? 3 : 1;
  static constexpr bool kSwz = kSwizzled<D> || D == 256;
  using S = std::conditional_t<kSwz, Swz<D>, Pad<D>>;
  static constexpr int kParts = (S::template bytes<kKeys>() + 1023) / 1024;  // loads of a tile
  static constexpr int kTileBytes = kParts * 1024;
  static constexpr int kFloats = kRows * D;  // a partial O
  // One workgroup per CU. Its waves have 48 to 128 KB of K and V under way, as much as
  // HBM needs: two per CU at D=64 read 5.4 TB/s where one reads 6.4 (B=32 H=32, up to
  // 8000 keys), and one after another they begin twice (19.8 us for 15.0 at B=8 H=16/4
  // D=64, 5 tokens, up to 4003 keys).
  static constexpr int kGrid = kCUs;
  // Whether a workgroup's waves meet in LDS: from a stretch of four blocks on, or two
  // where a part per block would be 64 or more for the items' mean (at D=128: 19.0 us
  // against 29.5 for one item of 625 blocks, 13.8 and 14.3 for 8 of 94; 13.3 and 12.6
  // for 32 of 19, 13.0 and 12.6 for 8 of 63).
  template <int TILES>
  __device__ __forceinline__ static bool joins(int stretch, int total, int items) {
    constexpr int kFrom = kLine<TILES> < 4 ? kLine<TILES> : 4;  // (a wave's stretch is a block below)
    return stretch >= kFrom || (stretch >= 2 && total / (64 / TILES) >= items);
  }
  static_assert(kWaves / 2 * kFloats * 4 <= kWaves * kTileBytes, "merge area exceeds the tiles");

  // The row and 16-byte chunk that lane `lane` of load u brings in.
  __device__ __forceinline__ static void place(int u, int lane, int& row, int& chunk) {
    if constexpr (kSwz) {
      row = S::kRowsPerInst * u + lane / S::kChunks;
      chunk = (lane % S::kChunks) ^ S::g(row);
    } else {
      const int p = u * 64 + lane, rho = p / Tile<D>::kStride;
      row = rho < kKeys ? perm16(rho) : 0;
      chunk = min(p - rho * Tile<D>::kStride, Tile<D>::kChunks - 1);
    }
  }
};

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
  bool by_item;  // the join's workgroups take an item each
  int runs;  // of 64 or 16 float4 columns in a tile's rows, slice (1 or 2) a join's workgroup
  int slice;
  float scale_log2, rescale, alibi_unit;  // (the last two in units of q . k)
  const float* alibi;
  Strides stq;
};

// A request's keys: [lo, len) are seen by some row, in key blocks first .. first + blocks - 1
// (at least one, so that requests without keys are items too).
struct Keys {
  int len, lo, first, blocks;
  __device__ __forceinline__ Keys(const PagedKernelArgs& a, int raw) {
    len = min(max(raw, 0), a.cap);
    lo = a.window > 0 ? max(0, len - a.N - a.window + 1) : 0;
    first = lo / kKeys;
    blocks = max(1, (len + kKeys - 1) / kKeys - first);
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
template <int D, int TILES>
struct Line {
  using T = Paged<D>;
  const PagedKernelArgs& a;
  const int lane;
  int lens, c0;      // kv_len of the requests c0 + lane (c0 < 0: none yet)
  int per, through;  // blocks of the requests up to (lane + 1) * per
  int lead;            // units of an item beside its blocks
  int total, stretch;  // all units, and those of a workgroup

  __device__ __forceinline__ Line(const PagedKernelArgs& a, int lane)
      : a(a), lane(lane), lens(0), c0(a.B > 64 ? -64 : 0), per((a.B + 63) / 64) {
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int c = lane * per + i;
      if (c < a.B) {
        lens = a.kv_len[c];
        mine += Keys(a, lens).blocks * a.items;
      }
    }
    through = wave_prefix(mine);
    total = __builtin_amdgcn_readlane(through, 63);
    stretch = (total + T::kGrid - 1) / T::kGrid;
    lead = stretch >= T::template kLine<TILES> ? 2 : 0;
    if (lead) {
      through += lead * min((lane + 1) * per, a.B) * a.items;
      total += lead * a.B * a.items;
      stretch = (total + T::kGrid - 1) / T::kGrid;
    }
  }
  __device__ __forceinline__ int units(const Keys& k) const { return k.blocks + lead; }
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
      const int x = c < min(a.B, (run + 1) * per) ? units(Keys(a, lens)) * a.items : 0;
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
    for (int i = lane; i < b; i += 64) sum += units(Keys(a, a.kv_len[i])) * a.items;
    return __builtin_amdgcn_readlane(wave_prefix(sum), 63);
  }
  __device__ __forceinline__ Keys keys(int b) {
    if ((unsigned)(b - c0) >= 64u) {
      c0 = b;
      lens = a.kv_len[min(b + lane, a.B - 1)];
    }
    return Keys(a, __builtin_amdgcn_readlane(lens, b - c0));
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

// A lane's row of an item's tile.
struct Row {
  bool ok;
  int hq, n;
  template <class Args>
  __device__ __forceinline__ Row(const Args& a, int hkv, int tile, int row) {
    const int rows = a.group * a.N, r = tile * kRows + row, rc = min(r, rows - 1);
    const int g = a.N == 1 ? rc : rc / a.N;
    ok = r < rows;
    hq = hkv * a.group + g;
    n = rc - g * a.N;
  }
};

// 16 bytes per lane from `from` to LDS at lds + byte_off + 16 * lane. STREAM: with
// the nontemporal hint. K and V that one row tile reads are read once, and hinted
// so they come at 6.5 TB/s (403 us at B=64 H=32/8 D=128, up to 16384 keys; 5.8 and
// 449 without); several tiles find them in L2, where the hint takes them out (32 us
// without it and 42 with it at B=4 H=32/8 D=128, 16 tokens, up to 8192 keys).
template <bool STREAM>
__device__ __forceinline__ void lds_direct(void* lds, const char* from, uint32_t byte_off) {
  auto* p = (__attribute__((address_space(3))) char*)lds + byte_off;
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)p, 16, 0, STREAM ? 2 : 0);
}

// 16 bytes each at two or four LDS addresses. In assembly, with their wait: ahead
// of an ordinary LDS read the compiler waits for every global_load_lds under way,
// whatever array it fills (of buffer loads to LDS it keeps them apart), which would
// hold K's products up for V's block.
typedef __attribute__((address_space(3))) const char lds_char;
__device__ __forceinline__ uint32_t lds_address(const char* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
__device__ __forceinline__ void lds_read(const uint32_t (&at)[2], u32x4 (&out)[2]) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(out[0]), "=&v"(out[1])
               : "v"(at[0]), "v"(at[1])
               : "memory");
}
__device__ __forceinline__ void lds_read(const uint32_t (&at)[4], u32x4 (&out)[4]) {
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\t"
               "ds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(out[0]), "=&v"(out[1]), "=&v"(out[2]), "=&v"(out[3])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
               : "memory");
}

// FULL: the head dim is the width. TILES: row tiles that waves abreast take. STREAM:
// there is one per kv head.
template <int D, bool BF, bool FULL, int TILES, bool STREAM>
__global__ __launch_bounds__(Paged<D>::kThreads, Paged<D>::kPerSimd) void paged_kernel(const PagedKernelArgs a) {
  using T = Paged<D>;
  using S = typename T::S;
  constexpr int kWaves = T::kWaves, kLine = T::template kLine<TILES>, kParts = T::kParts;
  __shared__ __align__(1024) char kt[kWaves * T::kTileBytes];
  __shared__ __align__(1024) char vt[kWaves * T::kTileBytes];
  __shared__ float2 ml[kWaves * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  const int wg = xcd_work_index(T::kGrid);
  const int on = wave / TILES, beside = wave % TILES;  // (of the waves on the line, of the tiles)
  Line<D, TILES> line(a, lane);
  if (wg == 0 && tid == 0) {
    a.sizes[0] = line.stretch;
    a.sizes[1] = line.total;
  }
  // The workgroup's stretch [wg0, wg1), and this wave's of it [pos, end): wave w
  // has block w of a stretch below kLine, else begins at floor(w * stretch / kLine).
  const int wg0 = wg * line.stretch, wg1 = min(wg0 + line.stretch, line.total);
  int4 owned = make_int4(0, 0, 0, 0);  // request, item, its start and units (none: 0)
  if (wg0 >= wg1) {
    if (lane == 0 && beside == 0) a.owned[wg * kLine + on] = owned;
    return;
  }
  const bool single = line.stretch < kLine;
  int pos = min(wg0 + (single ? on : on * line.stretch / kLine), wg1);
  const int end = min(wg0 + (single ? on + 1 : (on + 1) * line.stretch / kLine), wg1);
  int b, start;
  line.locate(min(pos, wg1 - 1), b, start);
  Keys keys = line.keys(b);
  int item = (min(pos, wg1 - 1) - start) / line.units(keys);
  start += item * line.units(keys);  // of the item, from here on
  const bool joins = T::template joins<TILES>(line.stretch, line.total, a.B * a.items);
  const bool join = joins && start <= wg0 && wg1 <= start + line.units(keys);
  if (!join && pos == end) {
    if (lane == 0 && beside == 0) a.owned[wg * kLine + on] = owned;
    return;
  }

  const uint32_t k_at = lds_address(kt) + wave * T::kTileBytes;
  char* const my_v = vt + wave * T::kTileBytes;
  const uint32_t page_bytes = 2u * (uint32_t)a.page_stride, row_bytes = 2u * (uint32_t)a.row_stride;
  const int page_mask = (1 << a.page_shift) - 1, dr = FULL ? D : a.dr, chunks = dr / 8;
  constexpr int kWaitOlder = 0x0F70 | (kParts & 15) | ((kParts >> 4) << 14);

  do {
    const int units = line.units(keys), from = pos - start, upto = min(from + end - pos, units);
    const int hkv = STREAM || a.n_groups == 1 ? item : item / a.n_groups;
    const int tile = STREAM ? 0 : (item - hkv * a.n_groups) * TILES + beside;
    // The blocks [j0, j1), and the page indices around them.
    const int j0 = keys.first + max(from - line.lead, 0);
    const bool some = keys.len > keys.lo && tile * kRows < a.group * a.N;  // (keys and rows)
    const int j1 = some ? keys.first + max(upto - line.lead, 0) : j0;
    const int* table = a.table + b * a.table_stride;
    const int last_page = max(keys.len - 1, 0) >> a.page_shift;
    int p0 = 0, held = 0;           // pages p0 .. p0 + 63 are in the lanes' `held`
    unsigned long long hidden = 0;  // of those, the ones outside the pool
    const char* base_k = (const char*)(a.k + hkv * a.head_stride);
    const char* base_v = (const char*)(a.v + hkv * a.head_stride);
    unsigned long long offs[kParts];  // of the loaded block's rows
    // The key that lane `ln` brings in with load u of block j.
    auto key_of = [&](int j, int u, int ln, int& chunk) {
      int r;
      T::place(u, ln, r, chunk);
      return min(max(j * kKeys + r, keys.lo), keys.len - 1);
    };
    auto fetch = [&](int j) {  // pages for block j
      p0 = max(j * kKeys, keys.lo) >> a.page_shift;
      const int page = table[min(p0 + lane, last_page)];
      wait_vmem();
      const bool ok = page >= 0 && page < a.pages;
      hidden = __ballot(!ok);
      held = ok ? page : 0;
    };
    auto place = [&](int j) {
      if ((min(j * kKeys + kKeys, keys.len) - 1) >> a.page_shift > p0 + 63) fetch(j);
      int ln = lane;
      asm("" : "+v"(ln));  // (the rows and columns are worked out again: registers are scarcer)
      constexpr int kAtOnce = kParts < 8 ? kParts : 8;
#pragma unroll
      for (int u0 = 0; u0 < kParts; u0 += kAtOnce) {
        uint32_t page[kAtOnce];
        int key[kAtOnce], chunk;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          key[i] = key_of(j, u0 + i, ln, chunk);
          page[i] = (uint32_t)__shfl(held, (key[i] >> a.page_shift) - p0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          (void)key_of(j, u0 + i, ln, chunk);
          // (past the head dim: unused)
          const uint32_t col = FULL || chunk < chunks ? 16u * (uint32_t)chunk : 0u;
          offs[u0 + i] = (unsigned long long)page[i] * page_bytes +
                         (unsigned long long)(uint32_t)(key[i] & page_mask) * row_bytes + col;
        }
      }
    };
    auto load = [&](char* array, const char* base) {
#pragma unroll
      for (int u = 0; u < kParts; ++u)
        lds_direct<STREAM>(array, base + offs[u], (uint32_t)(wave * T::kTileBytes + u * 1024));
    };

    // The way to the first loads is what a short call waits for: nothing that they
    // do not need comes before them. (q between K and V: the waits for K are its too.)
    if (j0 < j1) {
      fetch(j0);
      place(j0);
      load(kt, base_k);
    }
    int ln = lane;
    asm volatile("" : "+v"(ln));
    __builtin_amdgcn_sched_barrier(0);
    const int h = ln >> 5, l32 = ln & 31;
    LateArgs& qa = late_args();
    const Row row(qa, hkv, tile, l32);
    floatx16 oacc[D / 32];
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) oacc[cb] = zero16();
    float m_raw = -INFINITY, l = 0.f;
    if (j0 < j1) {
      const half_t* qrow = qa.q + b * qa.stq.b + row.hq * qa.stq.h + (size_t)row.n * qa.stq.n;
      half8 qb[D / 16];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        qb[kk] = as_half8(load16(qrow + kk * 16 + h * 8, FULL || kk * 16 + h * 8 < dr));
      const float slope = qa.alibi ? qa.alibi[row.hq] : 0.f;
      __builtin_amdgcn_sched_barrier(0);
      load(vt, base_v);
      // Keys [lo, hi) of this lane's row, and those that every row sees.
      const int at0 = keys.len - qa.N, at = at0 + row.n, window = qa.window;
      const int lo = window > 0 ? max(0, at - window + 1) : 0;
      const int hi = qa.causal ? min(keys.len, at + 1) : keys.len;
      const int all_lo = window > 0 ? max(0, keys.len - window) : 0;
      const int all_hi = qa.causal ? at0 + 1 : keys.len;
      typename S::Offsets off;
      off.init(ln, 0);
      const float alibi_raw = slope * qa.alibi_unit, c = qa.scale_log2, thr_raw = qa.rescale;
      for (int j = j0; j < j1; ++j) {
        const unsigned long long hide = hidden;  // (of block j's pages, from page hide0 on)
        const int hide0 = p0;
        __builtin_amdgcn_s_waitcnt(kWaitOlder);  // K's block is here, V's may be under way
        // (two sums, each product waiting for the one before of its own, where there
        // are registers for them)
        constexpr bool kTwo = D <= 128;
        floatx16 s = zero16(), s2 = zero16();
        constexpr int kRead = D % 64 == 0 ? 4 : 2;  // operands at a time
#pragma unroll
        for (int k0 = 0; k0 < D / 16; k0 += kRead) {
          uint32_t lds[kRead];
          u32x4 x[kRead];
#pragma unroll
          for (int i = 0; i < kRead; ++i) lds[i] = k_at + off.rd[k0 + i];
          lds_read(lds, x);
#pragma unroll
          for (int i = 0; i < kRead; i += 2) {
            s = mfma16<BF>(as_half8(x[i]), qb[k0 + i], s);
            floatx16& t = kTwo ? s2 : s;
            t = mfma16<BF>(as_half8(x[i + 1]), qb[k0 + i + 1], t);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        // (Loads behind the last block are one row again and again, and not used: a
        // branch around them would leave their number unknown, and every wait full.)
        if (j + 1 < j1) {
          place(j + 1);
        } else {
#pragma unroll
          for (int u = 0; u < kParts; ++u) offs[u] = 0;
        }
        load(kt, base_k);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] += kTwo ? s2[e] : 0.f;
        const int base = j * kKeys + 4 * h;
        if (alibi_raw != 0.f) {
          const float d0 = (float)(at - base);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[e] = fmaf(-alibi_raw, fabsf(d0 - (float)(8 * (e >> 2) + (e & 3))), s[e]);
        }
        if (j * kKeys < all_lo || (j + 1) * kKeys > all_hi) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = base + 8 * (e >> 2) + (e & 3);
            if (key < lo || key >= hi) s[e] = -INFINITY;
          }
        }
        if (hide) {  // pages outside the pool: their keys masked, their values zero
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = min(max(base + 8 * (e >> 2) + (e & 3), keys.lo), keys.len - 1);
            if ((hide >> ((key >> a.page_shift) - hide0)) & 1) s[e] = -INFINITY;
          }
        }
        float mloc = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mloc = fmaxf(mloc, s[e]);
        mloc = max_halves(mloc);
        if (__any(mloc > m_raw + thr_raw)) {
          const float m_new = fmaxf(m_raw, mloc);
          const float corr = m_raw == -INFINITY ? 0.f : fast_exp2((m_raw - m_new) * c);
          l *= corr;
#pragma unroll
          for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[cb][e] *= corr;
          m_raw = m_new;
        }
        // (s - m first: exact near the maximum, so that P is at most its scale's)
        const float m_use = m_raw == -INFINITY ? 0.f : m_raw;
        half8 pb[2], rest[2];
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = fast_exp2(fmaf(s[e] - m_use, c, (float)kPScale<BF>));
          ls[e & 3] += p;
          pb[e >> 3][e & 7] = to16<BF>(p);
          if constexpr (STREAM) rest[e >> 3][e & 7] = to16<BF>(p - from16<BF>(pb[e >> 3][e & 7]));
        }
        // (a block's sum at a time: a sum near 1 does not feel single weights below 2^-25)
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        __builtin_amdgcn_s_waitcnt(kWaitOlder);  // V's block is here, K's next may be under way
        if (hide) {
#pragma unroll 1
          for (int u = 0; u < kParts; ++u) {
            int chunk;
            if ((hide >> ((key_of(j, u, lane, chunk) >> a.page_shift) - hide0)) & 1)
              *reinterpret_cast<u32x4*>(my_v + u * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
          }
          wait_lds();
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int cb = 0; cb < D / 32; ++cb) {
            const half8 v = S::tr_operand(my_v, q, off, cb);
            oacc[cb] = mfma16<BF>(v, pb[q], oacc[cb]);
            if constexpr (STREAM) oacc[cb] = mfma16<BF>(v, rest[q], oacc[cb]);
          }
        wait_lds();
        load(vt, base_v);
      }
    }
    wait_vmem();

    // The rows' results, or the part's: unscaled O, maximum and sum. Part slots:
    // two of a wave, the first for the item that it does not begin and the second
    // for the one that it does; the first of its first wave for a workgroup's; the
    // block's position where no stretch is joined (a block is a part there).
    asm volatile("" : "+v"(ln));  // (addresses are worked out here, not kept through the loop)
    const int lh = ln >> 5, lr = ln & 31;
    LateArgs& ra = late_args();
    const float c = ra.scale_log2;
    const int n = upto - from;
    if (from == 0 && n > 0 && n < units) owned = make_int4(b, item, start, units);
    size_t slot = (joins ? 2 * (wg * kLine + on) + (from > 0 ? 0 : 1) : pos) * TILES + beside;
    half_t* orow = ra.o + b * ra.stq.b + row.hq * ra.stq.h + (size_t)row.n * ra.stq.n;
    // (a sum of 0: no key. NaN stays NaN, and does not say that there was none.)
    auto finish = [&](bool whole, float m, float sum) {
      if (!whole) ra.part_ml[slot * ra.part_rows + lr] = make_float2(m * c, sum);
      else if (ra.lse)
        ra.lse[((size_t)b * ra.Hq + row.hq) * ra.N + row.n] =
            sum == 0.f ? INFINITY : (m * c + __log2f(sum * kPUnit<BF>)) * kLn2;
    };
    // Columns col .. col + 3 (a row without keys: O = 0).
    auto put = [&](bool whole, float inv, int col, floatx4 v) {
      if (!whole) {
        *reinterpret_cast<floatx4*>(ra.part_o + (slot * ra.part_rows + lr) * D + col) = v;
      } else if (FULL || col < dr) {
        half4 o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = to16<BF>(v[e] * inv);
        *reinterpret_cast<half4*>(orow + col) = o4;
      }
    };
    if (!join) {
      const bool whole = n == units;
      const float sum = l + xor32(l), inv = sum > 0.f ? 1.f / sum : 0.f;
      if (row.ok && n > 0) {
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            put(whole, inv, 32 * cb + 8 * g + 4 * lh,
                floatx4{oacc[cb][4 * g], oacc[cb][4 * g + 1], oacc[cb][4 * g + 2], oacc[cb][4 * g + 3]});
        if (lh == 0) finish(whole, m_raw, sum);
      }
      pos += n;
      start += units;
      if (++item == a.items && pos < end) {
        if (++b == a.B) break;
        item = 0;
        keys = line.keys(b);
      }
      continue;
    }
    // One item: the waves' parts meet in LDS (the rows that there are), in the
    // accumulator's order: float4 (cb * 4 + g) * 64 + lane.
    if (wg1 - wg0 == units) owned.w = 0;
    if (lane == 0 && beside == 0) ra.owned[wg * kLine + on] = owned;
    __syncthreads();
    auto part_of = [&](int src) {
      return reinterpret_cast<float*>(src < kWaves / 2 ? kt : vt) + src % (kWaves / 2) * T::kFloats;
    };
    if (row.ok) {
#pragma unroll
      for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<floatx4*>(part_of(wave) + ((cb * 4 + g) * 64 + ln) * 4) =
              floatx4{oacc[cb][4 * g], oacc[cb][4 * g + 1], oacc[cb][4 * g + 2], oacc[cb][4 * g + 3]};
    }
    ml[wave * 64 + ln] = make_float2(m_raw, l);
    __syncthreads();
    if (!row.ok) return;
    float m_star = -INFINITY, l_star = 0.f, wk[kLine];
    const float2* const mine = ml + beside * 64;
#pragma unroll
    for (int k = 0; k < kLine; ++k) m_star = fmaxf(m_star, mine[k * TILES * 64 + ln].x);
#pragma unroll
    for (int k = 0; k < kLine; ++k) {
      const float2 x = mine[k * TILES * 64 + ln];
      wk[k] = x.x == -INFINITY ? 0.f : fast_exp2((x.x - m_star) * c);
      l_star += wk[k] * (x.y + mine[k * TILES * 64 + (ln ^ 32)].y);
    }
    const bool whole = wg1 - wg0 == units;
    const float inv = l_star > 0.f ? 1.f / l_star : 0.f;
    slot = 2 * (size_t)(wg * kLine) * TILES + beside;
    constexpr int kRuns = D / 8;  // float4 runs per lane, dealt to the waves
#pragma unroll
    for (int i = 0; i < (kRuns + kLine - 1) / kLine; ++i) {
      const int run = i * kLine + on;
      if (run >= kRuns) break;
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kLine; ++k)
        acc += *reinterpret_cast<const floatx4*>(part_of(k * TILES + beside) + (run * 64 + ln) * 4) * wk[k];
      put(whole, inv, 8 * run + 4 * lh, acc);
    }
    if (on == 0 && lh == 0) finish(whole, m_star, l_star);
    return;
  } while (pos < end);
  if (lane == 0 && beside == 0) late_args().owned[wg * kLine + on] = owned;
}

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
template <int D, bool BF, bool FULL, int TILES, int RUN>
__global__ __launch_bounds__(64 * kMergeWaves, 6) void paged_merge_kernel(const PagedKernelArgs a) {
  constexpr int kLine = Paged<D>::template kLine<TILES>;
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
    Line<D, TILES> line(a, lane);
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
         (Paged<D>::template joins<TILES>(stretch, total, a.B * a.items) && start == g0 * stretch &&
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
    if (Paged<D>::template joins<TILES>(stretch, total, a.B * a.items)) {
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
    constexpr int kSlots = Paged<D>::kGrid * kLine * 2;
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
      const Row row(a, hkv, tile, rr);
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (FULL || col < a.dr) {
        half4 o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = to16<BF>(acc[e] * inv);
        *reinterpret_cast<half4*>(a.o + b * a.stq.b + row.hq * a.stq.h + (size_t)row.n * a.stq.n + col) = o4;
      }
      if (col == 0 && a.lse)
        a.lse[((size_t)b * a.Hq + row.hq) * a.N + row.n] =
            l == 0.f ? INFINITY : (m + __log2f(l * kPUnit<BF>)) * kLn2;
    }
  }
}

}  // namespace

template <>
size_t paged_workspace_w<FA_WIDTH, FA_BF>(int rows) {
  constexpr size_t kAll = (size_t)Paged<FA_WIDTH>::kGrid * Paged<FA_WIDTH>::kWaves;
  return kAll * 2 * min(rows, kRows) * (FA_WIDTH * sizeof(float) + sizeof(float2)) +
         kAll * sizeof(int4) + 2 * sizeof(int);
}

template <>
hipError_t launch_paged_w<FA_WIDTH, FA_BF>(const PagedArgs& a) {
  constexpr int D = FA_WIDTH;
  PagedKernelArgs d{};
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
  d.part_rows = min(d.group * a.N, kRows);
  d.part_o = (float*)a.workspace;
  constexpr size_t kAll = (size_t)Paged<D>::kGrid * Paged<D>::kWaves;
  d.part_ml = (float2*)(d.part_o + kAll * 2 * d.part_rows * D);
  d.owned = (int4*)(d.part_ml + kAll * 2 * d.part_rows);
  d.sizes = (int*)(d.owned + kAll);
  const int n_tiles = (d.group * a.N + kRows - 1) / kRows;
  // Several row tiles per kv head go abreast, two or four, but where full tables are
  // 16 MB, which L2 holds anyway, and where a half of two pairs would be idle.
  const bool small = (long long)a.B * d.cap * a.Hkv * a.D * 4 <= 16 << 20;
  const int tiles = n_tiles == 1 || small || (D > 128 && n_tiles == 3) ? 1
                    : n_tiles == 2 || D > 128                           ? 2
                                                                        : 4;
  d.n_groups = (n_tiles + tiles - 1) / tiles;
  d.items = a.Hkv * d.n_groups;
  d.causal = a.causal;
  d.window = a.window < d.cap ? a.window : 0;  // (a wider one hides nothing)
  d.dr = a.D;
  d.scale_log2 = kLog2e * (a.scale > 0.f ? a.scale : 1.f / sqrtf((float)a.D));
  d.rescale = kPRescale<FA_BF> / d.scale_log2;
  d.alibi_unit = kLog2e / d.scale_log2;
  d.alibi = a.alibi;
  d.stq = make_strides(a.layout, a.Hq, a.N, a.D);
  // A join workgroup per item and run where these are at most half as many as the
  // list's (3.8 us against 4.8 at B=8 H=16/4 D=64, 5 tokens: 160 and 768 workgroups;
  // 4.6 against 6.1 at B=30 H=16/2 D=256: 480 and 1024); else the list, a shorter way to
  // the parts (4.3 against 7.8 at B=40 H=16/4 D=64, 4 tokens: 512 and 640; 6.5 against
  // 13.4 at B=100 H=16/2 D=256: 1024 and 1600), with two runs each (1.3 us less
  // than with one at B=250 H=32/4 D=128). The list too for items of one run, but for
  // up to four of them, whose parts can be many (at B=1 H=16/4 D=64: 4.2 us against
  // 4.9 at 4000 keys, 3.9 and 3.4 at 1000).
  const long long items = (long long)a.B * d.items;
  const int columns = d.part_rows * (D / 4);
  d.runs = (columns + 63) / 64;
  d.by_item = (d.runs > 1 || items <= 4) &&
              2 * items * d.runs * tiles <= Paged<D>::kGrid * ((d.runs * tiles + 1) / 2);
  // Of 16 columns where few workgroups would join many parts: 5.8 us for 9.0 at B=1 H=8/1
  // D=128, 20000 keys (4 workgroups, 16 with shorter runs).
  const bool narrow = d.by_item && items * d.runs * tiles <= 64;
  if (narrow) d.runs = (columns + 15) / 16;
  d.slice = d.by_item ? 1 : 2 * tiles;
  const unsigned slices = (unsigned)((d.runs * tiles + d.slice - 1) / d.slice);
  auto launch = [&](auto full, auto abreast, auto stream) {
    constexpr bool kFull = decltype(full)::value, kStream = decltype(stream)::value;
    constexpr int kTiles = decltype(abreast)::value;
    hipLaunchKernelGGL((paged_kernel<D, FA_BF, kFull, kTiles, kStream>), dim3(Paged<D>::kGrid),
                       dim3(Paged<D>::kThreads), 0, (hipStream_t)a.stream, d);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const auto merge = narrow ? paged_merge_kernel<D, FA_BF, kFull, kTiles, 16>
                              : paged_merge_kernel<D, FA_BF, kFull, kTiles, 64>;
    hipLaunchKernelGGL(merge,
                       dim3(d.by_item ? (unsigned)items : Paged<D>::kGrid, slices),
                       dim3(64 * kMergeWaves), 0, (hipStream_t)a.stream, d);
    return hipGetLastError();
  };
  auto by_tiles = [&](auto full) {
    using std::false_type, std::true_type;
    if (n_tiles == 1) return launch(full, std::integral_constant<int, 1>{}, true_type{});
    if (tiles == 1) return launch(full, std::integral_constant<int, 1>{}, false_type{});
    if constexpr (D <= 128)
      if (tiles == 4) return launch(full, std::integral_constant<int, 4>{}, false_type{});
    return launch(full, std::integral_constant<int, 2>{}, false_type{});
  };
  return a.D == D ? by_tiles(std::true_type{}) : by_tiles(std::false_type{});
}

}  // namespace fa
