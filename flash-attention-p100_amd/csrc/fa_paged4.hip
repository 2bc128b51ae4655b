// Attention of the newest tokens of each request over a paged cache in 4 bits. A row of
// K or V is codes of 4 bits (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) and a power
// of two per 32 of them, so a value is code * 2^(scale - 127). No counterpart in the
// reference, which has no cache.
//
// As in fa_paged.hip the key blocks of all requests lie on one line that the waves
// divide evenly, and the parts of an item meet in LDS and in paged_merge_kernel (few short
// items take a workgroup each, and meet in LDS alone). A
// wave's step is a block of 64 keys for RT tiles of 16 query rows, on
// v_mfma_f32_16x16x32_bf16: S^T = K Q^T, then O^T += V^T P^T. Every value of the cache is
// exact in bf16 (a sign, two bits and an exponent), whatever q's format, and
// v_cvt_scalef32_pk_bf16_fp4 makes two of them from a byte, scale included:
//   * K: a lane's codes are an MFMA operand as they lie (key lane % 16, a quarter of the
//     row), so they go from memory to registers and need no LDS;
//   * V: the second product runs over keys, so the values are written to LDS as bf16 and
//     come back transposed (ds_read_b64_tr_b16).
// q in fp16 has 11 bits: two bf16 numbers, exactly, and two products. The probabilities
// are two bf16 numbers (off by 2^-16), two products too. Sums of the rows are taken of the
// fp32 weights (by the matrix unit, of the rounded ones, the lse was off by 2^-9).
//
// Bound: HBM. 64 requests of 3300 to 16384 tokens, H=32/8 D=128 N=1 (684 MB): 116 us, 5.9
// TB/s, where the loads alone take 110, and 5 to join the parts. That took blocks loaded
// ahead of the one that is multiplied, at places held in scalar registers, with scales as
// whole words (145 us before: bytes are widened, and so waited for, at once); 16 waves of 32
// keys, with half the LDS each, took 124. Short lines are bound by latency: 3.5 us until a
// wave's first keys are there, then a block in 2.5 us (16 requests of 800 to 8192: 23 us,
// five blocks at most to a wave, 12 for their 77 MB alone; one of 1021: 6.6, and 3.4 to
// join). One conversion of a block serves two row tiles; four, with their sums, do not fit
// into registers (N=16 H=32/8: 186 us against 59).
#include "fa_paged.h"

namespace fa {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int DIM, bool OUT_BF, int RT>
struct Paged4 {
  static constexpr int kD = DIM, kTiles = 1, kRowTiles = RT, kRows = 16 * RT;
  static constexpr int kKeys = 64;
  static constexpr bool kBF = OUT_BF;
  static constexpr int kWaves = 8 / (DIM > 128 ? 2 : 1), kLine = kWaves;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kGrid = kCUs;
  static constexpr float kPUnit = 1.f, kPRescale = kRescaleLog2;
  static constexpr int kBlocks = DIM / 32;  // of a row, each with its scale
  static constexpr int kQ = OUT_BF ? 1 : 2;  // bf16 operands of q
  // LDS rows of V: eight 16-byte chunks in a row of keys, two of each, lie in 16 bank
  // groups (the row's chunks are 2 more than a multiple of 4).
  static constexpr int kStride = 2 * DIM + 32;
  static constexpr int kTileBytes = kKeys * kStride;
  static_assert(kRows * DIM * 4 <= kTileBytes, "a part exceeds the wave's tile");
  __device__ __forceinline__ static bool joins(int stretch, int total, int items) {
    constexpr int kFrom = kLine < 4 ? kLine : 4;
    return stretch >= kFrom || (stretch >= 2 && total / 64 >= items);
  }
};

struct Paged4Args : PagedKernelArgs {
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  long long scale_page, scale_head, scale_row;
  uint32_t code_bytes, scale_bytes;  // of a kv head's rows, first to last (PAGES > 0)
};

__device__ __forceinline__ floatx4 mfma_bf16(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The eight values of a dword of codes.
__device__ __forceinline__ half8 values(uint32_t codes, float scale) {
  const uint32_t r[4] = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  return as_half8(u32x4{r[0], r[1], r[2], r[3]});
}
// The scale that lies `at` bits up in a word: its bits moved to an exponent's place. (The
// conversion takes the exponent of its scale alone, whatever the sign and mantissa are.)
__device__ __forceinline__ float scale_of(uint32_t word, uint32_t at) {
  return __uint_as_float(__builtin_amdgcn_alignbit(word, word, (at + 9u) & 31u));
}

// The maximum over lanes l, l ^ 16, l ^ 32 and l ^ 48, which hold the same query row.
__device__ __forceinline__ float max_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// FULL: the head dim is the width (else 160, 192 or 224 of 256). PAGES: those of a tile of
// 16 keys. With 1 (pages of 16 rows or more) or 2 (of 8) a page's place is found once, in
// scalar registers, and a lane adds an offset of its own that never changes; 0: a key at a
// time. STREAM: one row tile reads the keys.
template <class T, bool FULL, int PAGES, bool STREAM>
__global__ __launch_bounds__(T::kThreads) void paged4_kernel(const Paged4Args a) {
  constexpr int D = T::kD, RT = T::kRowTiles, kWaves = T::kWaves, kLine = T::kLine;
  constexpr int kDwords = D / 32;  // of codes in a lane's quarter of a row
  constexpr int kKeys = T::kKeys, kKeyTiles = kKeys / 16, kScores = 4 * kKeyTiles;
  __shared__ __align__(1024) char vt[kWaves * T::kTileBytes];
  __shared__ float2 ml[RT * kWaves * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  const int wg = a.by_item ? (int)blockIdx.x : xcd_work_index(T::kGrid);
  const int l16 = lane & 15, g = lane >> 4;
  // by_item: an item to a workgroup, whose waves meet in LDS. Else the line.
  int b = a.by_item ? wg / a.items : 0, item = wg - b * a.items, start = 0;
  Keys<T> keys(a, a.by_item ? a.kv_len[b] : 0);
  Line<T> line = a.by_item ? Line<T>(a, lane, keys.blocks) : Line<T>(a, lane);
  if (!a.by_item && wg == 0 && tid == 0) {
    a.sizes[0] = line.stretch;
    a.sizes[1] = line.total;
  }
  const int wg0 = a.by_item ? 0 : wg * line.stretch, wg1 = min(wg0 + line.stretch, line.total);
  int4 owned = make_int4(0, 0, 0, 0);  // request, item, its start and units (none: 0)
  if (wg0 >= wg1) {
    if (lane == 0) a.owned[wg * kLine + wave] = owned;
    return;
  }
  const bool single = line.stretch < kLine;
  int pos = min(wg0 + (single ? wave : wave * line.stretch / kLine), wg1);
  const int end = min(wg0 + (single ? wave + 1 : (wave + 1) * line.stretch / kLine), wg1);
  if (!a.by_item) {
    line.locate(min(pos, wg1 - 1), b, start);
    keys = line.keys(b);
    item = (min(pos, wg1 - 1) - start) / line.units(keys);
    start += item * line.units(keys);  // of the item, from here on
  }
  const bool joins = a.by_item || T::joins(line.stretch, line.total, a.B * a.items);
  const bool join = joins && start <= wg0 && wg1 <= start + line.units(keys);
  if (!join && pos == end) {
    if (lane == 0) a.owned[wg * kLine + wave] = owned;
    return;
  }

  char* const my_v = vt + wave * T::kTileBytes;
  const uint32_t page_bytes = (uint32_t)a.page_stride, row_bytes = (uint32_t)a.row_stride;
  const uint32_t scale_page = (uint32_t)a.scale_page, scale_row = (uint32_t)a.scale_row;
  const int page_mask = (1 << a.page_shift) - 1, dr = FULL ? D : a.dr;

  do {
    const int units = line.units(keys), from = pos - start, upto = min(from + end - pos, units);
    const int hkv = a.n_groups == 1 ? item : item / a.n_groups;
    const int tile = item - hkv * a.n_groups;
    const int j0 = keys.first + max(from - line.lead, 0);
    const bool some = keys.len > keys.lo;
    const int j1 = some ? keys.first + max(upto - line.lead, 0) : j0;
    const int* table = a.table + b * a.table_stride;
    const int last_page = max(keys.len - 1, 0) >> a.page_shift;
    int p0 = 0, held = 0, next = 0;  // pages p0 .. p0 + 63 are in the lanes' `held`, then 64 more
    unsigned long long hidden = 0;   // of those held, the ones outside the pool
    const uint8_t* const base_k = (const uint8_t*)a.k + hkv * a.head_stride;
    const uint8_t* const base_v = (const uint8_t*)a.v + hkv * a.head_stride;
    // (the scales of a kv head begin anywhere in a word: with PAGES from the word on)
    const uint8_t* base_ks = a.k_scale + hkv * a.scale_head;
    const uint8_t* base_vs = a.v_scale + hkv * a.scale_head;
    const uint32_t sub_k = PAGES ? (uint32_t)((uintptr_t)base_ks & 3) : 0u;
    const uint32_t sub_v = PAGES ? (uint32_t)((uintptr_t)base_vs & 3) : 0u;
    base_ks -= sub_k;
    base_vs -= sub_v;
    const rsrc_t codes_k = make_rsrc(base_k, a.code_bytes), codes_v = make_rsrc(base_v, a.code_bytes);
    const rsrc_t scales_k = make_rsrc(base_ks, a.scale_bytes), scales_v = make_rsrc(base_vs, a.scale_bytes);
    auto hold = [&](int page) {
      const bool ok = page >= 0 && page < a.pages;
      hidden = __ballot(!ok);
      held = ok ? page : 0;
      next = table[min(p0 + 64 + lane, last_page)];
    };
    auto fetch = [&](int j) {  // pages for block j
      p0 = max(j * kKeys, keys.lo) >> a.page_shift;
      hold(table[min(p0 + lane, last_page)]);
    };
    auto place = [&](int j) {
      if ((min(j * kKeys + kKeys, keys.len) - 1) >> a.page_shift <= p0 + 63) return;
      if (PAGES > 0 && (j * kKeys) >> a.page_shift == p0 + 64) {  // (in order: they have been asked for)
        p0 += 64;
        hold(next);
      } else {
        fetch(j);
      }
    };
    // A block in registers: a quarter of a row in each of its tiles of 16 keys, K's of key
    // lane % 16 (as the product takes it), V's of key lane / 4 (as it lies in memory). Scales
    // come as the words that hold them: a byte would be widened, and waited for, at once.
    constexpr int kScales = D == 96 || (D == 256 && !FULL) ? 2 : 1;
    constexpr int kBits = PAGES == 0 ? kScales : 0;  // (rows anywhere: their scales' bits too)
    struct Codes {
      uint32_t c[kDwords], s[kScales], bit[kBits + 1];
    };
    // Where a lane's quarter `part` of key `key` of a tile lies, and its scales: the words
    // that hold them and the bits that they begin at.
    struct Place {
      uint32_t code, scale[kScales], bit[kScales];
      int second;        // the page of a tile that the key is in
      uint32_t back;     // how far before its first scale the row begins, or 2 bytes
      bool there, both;  // whether the quarter begins, and ends, within the head dim
      __device__ __forceinline__ Place(int key, int part, uint32_t row_bytes, uint32_t scale_row, int dr,
                                       uint32_t sub)
          : second(0), back(part ? 2u : 0u) {
        if (PAGES == 2) {
          second = key >> 3;
          key &= 7;
        }
        if (PAGES == 0) key = 0;  // (rows are found one by one)
        there = FULL || 64 * part < dr;
        both = FULL || 64 * part + 32 < dr;
        code = (uint32_t)key * row_bytes + 4u * kDwords * (there ? part : 0);
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
          const int block = !there ? 0 : D == 256 ? 2 * part + (both ? i : 0) : (kDwords * part + 2 * i) / 4;
          const uint32_t at = (uint32_t)key * scale_row + (uint32_t)block + sub;
          scale[i] = PAGES == 0 ? at : at & ~3u;
          bit[i] = 8 * (at & 3u);
        }
      }
      // The scales of a quarter's eighths, of 8 values each. (Values past the head dim meet
      // zeros of q: a finite scale.)
      __device__ __forceinline__ void sizes(const Codes& x, int part, float (&size)[kDwords]) const {
        float two[2];
#pragma unroll
        for (int i = 0; i < kScales; ++i) two[i] = scale_of(x.s[i], PAGES == 0 ? x.bit[i % (kBits + 1)] : bit[i]);
        if constexpr (kScales == 1) two[1] = D == 256 ? scale_of(x.s[0], (PAGES == 0 ? x.bit[0] : bit[0]) + 8) : two[0];
        if constexpr (!FULL) {
          two[0] = there ? two[0] : 1.f;
          two[1] = both ? two[1] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < kDwords; ++i) {
          if constexpr (D == 96) size[i] = i == 0 || (i == 1 && part != 1) ? two[0] : two[1];
          else size[i] = two[D == 256 ? i / 4 : 0];
        }
      }
    };
    const Place place_k(l16, g, row_bytes, scale_row, dr, sub_k);
    const Place place_v(lane >> 2, lane & 3, row_bytes, scale_row, dr, sub_v);
    // Where a quarter comes from: with PAGES a buffer of the kv head's rows, the tile's place
    // in it (uniform) and the lane's in the tile; else the row's own addresses.
    auto fill = [&](Codes& x, const Place& at, auto&& code16, auto&& scale_word) {
      if constexpr (D == 256) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 v = code16(FULL || at.both ? 16 * h : 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) x.c[(4 * h + i) % kDwords] = v[i];
        }
      } else {
        const u32x4 v = code16(0);  // (of less where a quarter is less)
#pragma unroll
        for (int i = 0; i < kDwords; ++i) x.c[i] = v[i % 4];
      }
#pragma unroll
      for (int i = 0; i < kScales; ++i) x.s[i] = scale_word(i, x);
    };
    auto load_tile = [&](Codes& x, rsrc_t codes, rsrc_t scales, const Place& at, uint32_t to, uint32_t sto,
                         uint32_t lane_to, uint32_t lane_sto) {
      constexpr int kAux = STREAM ? 2 : 0;  // (the nontemporal hint)
      fill(x, at,
           [&](int off) {
             const uint32_t v = at.code + lane_to;
             if constexpr (kDwords == 1) return u32x4{__builtin_amdgcn_raw_buffer_load_b32(codes, v, to, kAux), 0, 0, 0};
             if constexpr (kDwords == 2) {
               const auto r = __builtin_amdgcn_raw_buffer_load_b64(codes, v, to, kAux);
               return u32x4{r[0], r[1], 0, 0};
             }
             if constexpr (kDwords == 3) {
               const auto r = __builtin_amdgcn_raw_buffer_load_b96(codes, v, to, kAux);
               return u32x4{r[0], r[1], r[2], 0};
             }
             return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(codes, v + off, to, kAux));
           },
           [&](int i, Codes&) { return __builtin_amdgcn_raw_buffer_load_b32(scales, at.scale[i] + lane_sto, sto, 0); });
    };
    auto load_row = [&](Codes& x, const uint8_t* row, const uint8_t* scales, const Place& at) {
      const uint8_t* const from = row + at.code;
      fill(x, at,
           [&](int off) {
             u32x4 v = {0u, 0u, 0u, 0u};
             if constexpr (kDwords < 4) __builtin_memcpy(&v, __builtin_assume_aligned(from, 4), 4 * kDwords);
             else v = *reinterpret_cast<const u32x4*>(from + off);
             return v;
           },
           [&](int i, Codes& x) {
             const uint8_t* word = scales + at.scale[i];
             uint32_t before = (uint32_t)((uintptr_t)word & 3u);
             // (Two scales of which the second lies behind the word: a word from an odd byte
             // on, within the row. Such words alone take longer, 53.7 us for 51 at B=16 H=32/8
             // N=1 D=256, 4000 keys in pages of 4; each scale by its own word spills more.)
             if constexpr (D == 256 && FULL)
               if (before == 3) before = at.back;
             x.bit[i % (kBits + 1)] = 8u * before;
             uint32_t w;
             __builtin_memcpy(&w, word - before, 4);
             return w;
           });
    };
    // Block j's K or V, or, where it is not live, a row of its memory, not used: a branch
    // around the loads would leave their number unknown, and every wait full.
    auto load_tiles = [&](Codes (&k)[kKeyTiles], Codes (&v)[kKeyTiles], int j, bool live) {
      // (a tile behind the last key: some of its rows' memory, masked)
      auto place_of = [&](int key, uint32_t& to, uint32_t& sto) {
        const int i = max((min(key, keys.len - 1) >> a.page_shift) - p0, 0);
        const uint32_t page = live ? (uint32_t)__builtin_amdgcn_readlane(held, i) : 0u;
        const uint32_t row = live && PAGES == 1 ? (uint32_t)(key & page_mask) : 0u;
        to = page * page_bytes + row * row_bytes;
        sto = page * scale_page + row * scale_row;
      };
      uint32_t to[kKeyTiles], sto[kKeyTiles], to2[kKeyTiles], sto2[kKeyTiles];
#pragma unroll
      for (int t = 0; t < kKeyTiles; ++t) {
        place_of(j * kKeys + 16 * t, to[t], sto[t]);
        if constexpr (PAGES == 2) place_of(j * kKeys + 16 * t + 8, to2[t], sto2[t]);
        else to2[t] = to[t], sto2[t] = sto[t];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int t = 0; t < kKeyTiles; ++t) {
          const Place& at = half ? place_v : place_k;
          const uint32_t lane_to = at.second ? to2[t] : to[t], lane_sto = at.second ? sto2[t] : sto[t];
          load_tile(half ? v[t] : k[t], half ? codes_v : codes_k, half ? scales_v : scales_k, at,
                    PAGES == 1 ? to[t] : 0u, PAGES == 1 ? sto[t] : 0u, PAGES == 1 ? 0u : lane_to,
                    PAGES == 1 ? 0u : lane_sto);
        }
    };
    auto load_rows = [&](Codes (&x)[kKeyTiles], const uint8_t* base, const uint8_t* scales, int key, const Place& at,
                         int j, bool live) {
#pragma unroll
      for (int t = 0; t < kKeyTiles; ++t) {
        const int k = min(max(j * kKeys + 16 * t + key, keys.lo), keys.len - 1);
        const uint32_t page = live ? (uint32_t)__shfl(held, (k >> a.page_shift) - p0) : 0u;
        const uint32_t row = live ? (uint32_t)(k & page_mask) : 0u;
        load_row(x[t], base + (unsigned long long)page * page_bytes + (unsigned long long)row * row_bytes,
                 scales + (unsigned long long)page * scale_page + (unsigned long long)row * scale_row, at);
      }
    };
    Codes kc[kKeyTiles], vc[kKeyTiles];
    auto load_both = [&](int j, bool live) {
      if (live) place(j);
      if constexpr (PAGES > 0) {
        load_tiles(kc, vc, j, live);
      } else {
        load_rows(kc, base_k, base_ks, l16, place_k, j, live);
        load_rows(vc, base_v, base_vs, lane >> 2, place_v, j, live);
      }
    };

    float m_raw[RT], l[RT];
    floatx4 oacc[RT][D / 16];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_raw[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) oacc[rt][c] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const float c = late_args().scale_log2;
    if (j0 < j1) {
      fetch(j0);
      LateArgs& qa = late_args();
      half8 q[RT][T::kQ][kDwords];
      float slope[RT];
      int row_n[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const Row<T::kRows> row(qa, hkv, tile, 16 * rt + l16);
        const half_t* qrow = qa.q + b * qa.stq.b + row.hq * qa.stq.h + (size_t)row.n * qa.stq.n;
        row_n[rt] = row.n;
        slope[rt] = qa.alibi ? qa.alibi[row.hq] * qa.alibi_unit : 0.f;
#pragma unroll
        for (int i = 0; i < kDwords; ++i) {
          const int d = D / 4 * g + 8 * i;
          q[rt][0][i] = as_half8(load16(qrow + d, FULL || d < dr));
        }
      }
      load_both(j0, true);
      // (q is waited for here, behind the loads of K and V: left to its first use, in the loop,
      // it would be waited for there, and with it all loads of every block)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < kDwords; ++i) {
          asm volatile("" : "+v"(q[rt][0][i]));
          if constexpr (!T::kBF) {
            const half8 x = q[rt][0][i];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float f = (float)x[e];
              q[rt][0][i][e] = to16<true>(f);
              const float rest = f - from16<true>(q[rt][0][i][e]);
              q[rt][T::kQ - 1][i][e] = to16<true>(__builtin_isfinite(f) ? rest : 0.f);
            }
          }
        }
      const int at0 = keys.len - qa.N, window = qa.window;
      const int all_lo = window > 0 ? max(0, keys.len - window) : 0;
      const int all_hi = qa.causal ? at0 + 1 : keys.len;
      const bool causal = qa.causal, biased = qa.alibi != nullptr;
      const float thr_raw = qa.rescale;
      for (int j = j0; j < j1; ++j) {
        const unsigned long long hide = hidden;  // (of block j's pages, from page hide0 on)
        const int hide0 = p0;
        floatx4 s[RT][kKeyTiles];
#pragma unroll
        for (int t = 0; t < kKeyTiles; ++t) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
          float size[kDwords];
          place_k.sizes(kc[t], g, size);
#pragma unroll
          for (int i = 0; i < kDwords; ++i) {
            const half8 k = values(kc[t].c[i], size[i]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int x = 0; x < T::kQ; ++x) s[rt][t] = mfma_bf16(k, q[rt][x][i], s[rt][t]);
          }
        }
        // V's block as bf16 to LDS; values of keys that no row sees become zero.
        const bool part = j * kKeys < keys.lo || j * kKeys + kKeys > keys.len || hide;
#pragma unroll
        for (int t = 0; t < kKeyTiles; ++t) {
          const int key = 16 * t + (lane >> 2);
          if (part) {
            const int x = j * kKeys + key, y = min(max(x, keys.lo), keys.len - 1);
            if (x != y || ((hide >> ((y >> a.page_shift) - hide0)) & 1)) {
#pragma unroll
              for (int i = 0; i < kDwords; ++i) vc[t].c[i] = 0u;
#pragma unroll
              for (int i = 0; i < kScales; ++i) vc[t].s[i] = 0u;
            }
          }
          float size[kDwords];
          place_v.sizes(vc[t], lane & 3, size);
          char* to = my_v + key * T::kStride + 16 * kDwords * (lane & 3);
#pragma unroll
          for (int i = 0; i < kDwords; ++i)
            *reinterpret_cast<half8*>(to + 16 * i) =
                values(vc[t].c[i], size[i]);
        }
        const bool more = j + 1 < j1;
        load_both(more ? j + 1 : j, more);
        const int base = j * kKeys + 4 * g;  // key of s[.][t][r]: base + 16 t + r
        const bool edge = j * kKeys < all_lo || j * kKeys + kKeys > all_hi;
        half8 pb[RT][kKeyTiles / 2], rest[RT][kKeyTiles / 2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int at = at0 + row_n[rt];
          if (biased) {
            const float d0 = (float)(at - base);
#pragma unroll
            for (int e = 0; e < kScores; ++e)
              s[rt][e >> 2][e & 3] =
                  fmaf(-slope[rt], fabsf(d0 - (float)(16 * (e >> 2) + (e & 3))), s[rt][e >> 2][e & 3]);
          }
          if (edge) {
            const int lo = window > 0 ? max(0, at - window + 1) : 0;
            const int hi = causal ? min(keys.len, at + 1) : keys.len;
#pragma unroll
            for (int e = 0; e < kScores; ++e) {
              const int key = base + 16 * (e >> 2) + (e & 3);
              if (key < lo || key >= hi) s[rt][e >> 2][e & 3] = -INFINITY;
            }
          }
          if (hide) {
#pragma unroll
            for (int e = 0; e < kScores; ++e) {
              const int key = min(max(base + 16 * (e >> 2) + (e & 3), keys.lo), keys.len - 1);
              if ((hide >> ((key >> a.page_shift) - hide0)) & 1) s[rt][e >> 2][e & 3] = -INFINITY;
            }
          }
          float mloc = s[rt][0][0];
#pragma unroll
          for (int e = 1; e < kScores; ++e) mloc = fmaxf(mloc, s[rt][e >> 2][e & 3]);
          mloc = max_quarters(mloc);
          if (__any(mloc > m_raw[rt] + thr_raw)) {
            const float m_new = fmaxf(m_raw[rt], mloc);
            const float corr = m_raw[rt] == -INFINITY ? 0.f : fast_exp2((m_raw[rt] - m_new) * c);
            l[rt] *= corr;
#pragma unroll
            for (int cb = 0; cb < D / 16; ++cb) oacc[rt][cb] *= corr;
            m_raw[rt] = m_new;
          }
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
          const float m_c = m_raw[rt] == -INFINITY ? 0.f : m_raw[rt] * c;
#pragma unroll
          for (int e = 0; e < kScores; ++e) {
            const float p = fast_exp2(fmaf(s[rt][e >> 2][e & 3], c, -m_c));
            ls[e & 3] += p;
            const half_t p16 = to16<true>(p);
            pb[rt][e >> 3][e & 7] = p16;
            rest[rt][e >> 3][e & 7] = to16<true>(p - from16<true>(p16));
          }
          l[rt] += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        }
        // (row 4 g + t of 16 keys at columns 4 a .. 4 a + 3 of 16, lane = 16 g + 4 t + a)
        const half_t* from_v =
            reinterpret_cast<const half_t*>(my_v + (4 * g + (l16 >> 2)) * T::kStride + 8 * (l16 & 3));
#pragma unroll
        for (int u = 0; u < kKeyTiles / 2; ++u)
#pragma unroll
          for (int cb = 0; cb < D / 16; ++cb) {
            const half4 lo = lds_read_tr(from_v + 32 * u * (T::kStride / 2) + 16 * cb);
            const half4 hi = lds_read_tr(from_v + (32 * u + 16) * (T::kStride / 2) + 16 * cb);
            const half8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              oacc[rt][cb] = mfma_bf16(v, pb[rt][u], oacc[rt][cb]);
              oacc[rt][cb] = mfma_bf16(v, rest[rt][u], oacc[rt][cb]);
            }
          }
      }
    }

    // The rows' results, or the part's (slots as in fa_paged.hip).
    LateArgs& ra = late_args();
    const int n = upto - from;
    if (from == 0 && n > 0 && n < units) owned = make_int4(b, item, start, units);
    size_t slot = joins ? 2 * (wg * kLine + wave) + (from > 0 ? 0 : 1) : pos;
    // (a sum of 0: no key. NaN stays NaN, and does not say that there was none.)
    auto finish = [&](const Row<T::kRows>& row, bool whole, int lr, float m, float sum) {
      if (!whole) ra.part_ml[slot * ra.part_rows + lr] = make_float2(m * c, sum);
      else if (ra.lse)
        ra.lse[((size_t)b * ra.Hq + row.hq) * ra.N + row.n] =
            sum == 0.f ? INFINITY : (m * c + __log2f(sum)) * kLn2;
    };
    auto put = [&](const Row<T::kRows>& row, bool whole, int lr, float inv, int col, floatx4 v) {
      if (!whole) {
        *reinterpret_cast<floatx4*>(ra.part_o + (slot * ra.part_rows + lr) * D + col) = v;
      } else if (FULL || col < dr) {
        half_t* orow = ra.o + b * ra.stq.b + row.hq * ra.stq.h + (size_t)row.n * ra.stq.n;
        half4 o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = to16<T::kBF>(v[e] * inv);
        *reinterpret_cast<half4*>(orow + col) = o4;
      }
    };
    if (!join) {
      const bool whole = n == units;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int lr = 16 * rt + l16;
        const Row<T::kRows> row(ra, hkv, tile, lr);
        float sum = l[rt] + __shfl_xor(l[rt], 16);
        sum += xor32(sum);
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        if (!row.ok || n <= 0) continue;
#pragma unroll
        for (int cb = 0; cb < D / 16; ++cb) put(row, whole, lr, inv, 16 * cb + 4 * g, oacc[rt][cb]);
        if (g == 0) finish(row, whole, lr, m_raw[rt], sum);
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
    // One item: the waves' parts meet in LDS, in the accumulator's order: float4 (rt * D / 16
    // + cb) * 64 + lane.
    const bool whole = wg1 - wg0 == units;
    if (whole) owned.w = 0;
    if (lane == 0 && !ra.by_item) ra.owned[wg * kLine + wave] = owned;
    slot = 2 * (size_t)(wg * kLine);
    constexpr int kRuns = D / 16;
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int cb = 0; cb < kRuns; ++cb)
        *reinterpret_cast<floatx4*>(my_v + ((rt * kRuns + cb) * 64 + lane) * 16) = oacc[rt][cb];
      ml[(rt * kWaves + wave) * 64 + lane] = make_float2(m_raw[rt], l[rt]);
    }
    __syncthreads();
#pragma unroll 1
    for (int task = wave; task < RT * kRuns; task += kLine) {
      const int rt = task / kRuns, cb = task % kRuns;
      const float2* const mine = ml + rt * kWaves * 64;
      float m_star = -INFINITY, l_star = 0.f;
#pragma unroll
      for (int k = 0; k < kLine; ++k) m_star = fmaxf(m_star, mine[k * 64 + lane].x);
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kLine; ++k) {
        const float2* const x = mine + k * 64 + l16;
        const float wk = x->x == -INFINITY ? 0.f : fast_exp2((x->x - m_star) * c);
        l_star += wk * ((x[0].y + x[16].y) + (x[32].y + x[48].y));
        acc += *reinterpret_cast<const floatx4*>(vt + k * T::kTileBytes + (task * 64 + lane) * 16) * wk;
      }
      const int lr = 16 * rt + l16;
      const Row<T::kRows> row(ra, hkv, tile, lr);
      if (row.ok) {
        put(row, whole, lr, l_star > 0.f ? 1.f / l_star : 0.f, 16 * cb + 4 * g, acc);
        if (cb == 0 && g == 0) finish(row, whole, lr, m_star, l_star);
      }
    }
    return;
  } while (pos < end);
  if (lane == 0) late_args().owned[wg * kLine + wave] = owned;
}

// Row tiles that a wave takes: one or two.
template <int D, bool BF, class F>
auto by_row_tiles(int rows, const F& f) {
  if (rows <= 16) return f(Paged4<D, BF, 1>{});
  return f(Paged4<D, BF, 2>{});
}

}  // namespace

template <>
size_t paged4_workspace_w<FA_WIDTH, FA_BF>(int rows) {
  return by_row_tiles<FA_WIDTH, FA_BF>(rows, [&](auto t) { return paged_workspace<decltype(t)>(rows); });
}

template <>
hipError_t launch_paged4_w<FA_WIDTH, FA_BF>(const PagedArgs& a) {
  return by_row_tiles<FA_WIDTH, FA_BF>(a.Hq / a.Hkv * a.N, [&](auto t) {
    using T = decltype(t);
    Paged4Args d{};
    paged_args<T>(d, a);
    d.k_scale = a.scales.k;
    d.v_scale = a.scales.v;
    d.scale_page = a.scales.page_stride;
    d.scale_head = a.scales.head_stride;
    d.scale_row = a.scales.row_stride;
    // Tiles go by 32-bit places in a kv head's rows, and by words of scales that begin at the
    // same bits in every tile (a lane of width 256 takes two scales, of one word: from an even
    // byte). Else row by row, by words that hold each row's scales wherever they begin.
    const auto& sc = a.scales;
    const long long code_bytes = (a.pool.pages - 1LL) * a.pool.page_stride +
                                 ((1LL << a.pool.page_shift) - 1) * a.pool.row_stride + a.D / 2;
    const long long scale_bytes = (a.pool.pages - 1LL) * sc.page_stride +
                                  ((1LL << a.pool.page_shift) - 1) * sc.row_stride + a.D / 32;
    const uintptr_t odd = (uintptr_t)sc.k | (uintptr_t)sc.v | (uintptr_t)sc.head_stride | (uintptr_t)sc.row_stride;
    const bool words = sc.page_stride % 4 == 0 && (a.D != 256 || odd % 2 == 0);
    const bool near = code_bytes < 1LL << 32 && scale_bytes < (1LL << 32) - 8;
    const int pages = !words || !near ? 0 : a.pool.page_shift >= 4 ? 1 : a.pool.page_shift == 3 ? 2 : 0;
    if (pages > 0) {
      d.code_bytes = (uint32_t)code_bytes;
      d.scale_bytes = (uint32_t)(scale_bytes + 6) & ~3u;  // (of whole words, from the first's)
    }
    // Where a table holds two blocks of a request for each of a workgroup's waves at most, and
    // the card has a CU for every item: an item to a workgroup, and no parts to join. (It is the
    // table that counts, 1024 tokens at D <= 128 and 512 above: lengths are the device's. H=16/8
    // D=128, us with the call's host, against the line: one request of 200 keys 7.9 and 10.6, of
    // 1021 10.8 and 11.6, of 1500 13.3 and 10.9; 32 of 1000 13.2 and 17.8, 128 of 500 34.7
    // and 26.0.)
    const long long items = (long long)a.B * d.items;
    const int most = d.window > 0 ? min(d.cap, d.window + a.N + T::kKeys) : d.cap;
    d.by_item = items <= kCUs && most <= 2 * T::kLine * T::kKeys;
    auto launch = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      constexpr bool kStream = T::kRowTiles == 1;
      const auto kernel = pages == 1   ? paged4_kernel<T, kFull, 1, kStream>
                          : pages == 2 ? paged4_kernel<T, kFull, 2, kStream>
                                       : paged4_kernel<T, kFull, 0, kStream>;
      hipLaunchKernelGGL(kernel, dim3(d.by_item ? (unsigned)items : T::kGrid), dim3(T::kThreads), 0,
                         (hipStream_t)a.stream, d);
      const hipError_t e = hipGetLastError();
      return e != hipSuccess || d.by_item ? e : launch_paged_join<T, kFull>(d, (hipStream_t)a.stream);
    };
    if constexpr (T::kD == 256)
      if (a.D != T::kD) return launch(std::false_type{});
    return launch(std::true_type{});
  });
}

}  // namespace fa
