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
#include "fa_paged.h"

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

template <int D, bool BF, int TILES>
struct Paged {
  static constexpr int kD = D, kTiles = TILES, kRows = fa::kRows, kKeys = fa::kKeys;
  static constexpr bool kBF = BF;
  static constexpr float kPUnit = fa::kPUnit<BF>, kPRescale = fa::kPRescale<BF>;
  static constexpr int kWaves = D > 128 ? 4 : 8;
  static constexpr int kThreads = 64 * kWaves;
  // Row tiles of a kv head that waves abreast take, over the same keys, and the waves
  // of each: what one brings in the others find in L2. (In all 113 us for 146 at B=20
  // H=64/8 D=128, 7 tokens, up to 8000 keys, and 208 for 296 at D=256; tiles apart on
  // the line read from HBM each, and are better where L2 holds all: 14.1 for 14.6 at
  // B=1 H=64/8 D=128, 5 tokens, 2000 keys.)
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
  __device__ __forceinline__ static bool joins(int stretch, int total, int items) {
    constexpr int kFrom = kLine < 4 ? kLine : 4;  // (a wave's stretch is a block below)
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
__global__ __launch_bounds__((Paged<D, BF, TILES>::kThreads), (Paged<D, BF, TILES>::kPerSimd)) void paged_kernel(
    const PagedKernelArgs a) {
  using T = Paged<D, BF, TILES>;
  using S = typename T::S;
  constexpr int kWaves = T::kWaves, kLine = T::kLine, kParts = T::kParts;
  __shared__ __align__(1024) char kt[kWaves * T::kTileBytes];
  __shared__ __align__(1024) char vt[kWaves * T::kTileBytes];
  __shared__ float2 ml[kWaves * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  const int wg = xcd_work_index(T::kGrid);
  const int on = wave / TILES, beside = wave % TILES;  // (of the waves on the line, of the tiles)
  Line<T> line(a, lane);
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
  Keys<T> keys = line.keys(b);
  int item = (min(pos, wg1 - 1) - start) / line.units(keys);
  start += item * line.units(keys);  // of the item, from here on
  const bool joins = T::joins(line.stretch, line.total, a.B * a.items);
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
    const Row<kRows> row(qa, hkv, tile, l32);
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

}  // namespace

template <>
size_t paged_workspace_w<FA_WIDTH, FA_BF>(int rows) {
  return paged_workspace<Paged<FA_WIDTH, FA_BF, 1>>(rows);
}

template <>
hipError_t launch_paged_w<FA_WIDTH, FA_BF>(const PagedArgs& a) {
  constexpr int D = FA_WIDTH;
  const int n_tiles = (a.Hq / a.Hkv * a.N + kRows - 1) / kRows;
  // Several row tiles per kv head go abreast, two or four, but where full tables are
  // 16 MB, which L2 holds anyway, and where a half of two pairs would be idle.
  const bool small =
      (long long)a.B * (a.table_width << a.pool.page_shift) * a.Hkv * a.D * 4 <= 16 << 20;
  const int tiles = n_tiles == 1 || small || (D > 128 && n_tiles == 3) ? 1
                    : n_tiles == 2 || D > 128                           ? 2
                                                                        : 4;
  auto launch = [&](auto full, auto abreast, auto stream) {
    constexpr bool kFull = decltype(full)::value, kStream = decltype(stream)::value;
    constexpr int kTiles = decltype(abreast)::value;
    using T = Paged<D, FA_BF, kTiles>;
    PagedKernelArgs d{};
    paged_args<T>(d, a);
    hipLaunchKernelGGL((paged_kernel<D, FA_BF, kFull, kTiles, kStream>), dim3(T::kGrid),
                       dim3(T::kThreads), 0, (hipStream_t)a.stream, d);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_paged_join<T, kFull>(d, (hipStream_t)a.stream);
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
