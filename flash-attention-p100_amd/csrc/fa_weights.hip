// The weight that each key of a paged cache gets from the newest rows of its request,
// given the rows' lse: w[key, kv head] += sum over the rows that see the key and the
// query heads of the group of exp(score - lse). (What eviction by accumulated attention
// goes by: fa_evict.hip.) No counterpart in the reference, which has no cache.
//
// The lse is known, so keys do not depend on each other: the blocks of 64 keys of all
// requests and kv heads lie on one line that the waves divide evenly (as in fa_paged.hip), a
// wave holds a block of K as operands and goes over all rows of the kv head, 16 at a time, on
// v_mfma_f32_16x16x32, S = Q K^T: a lane has one key of a tile, so the rows' weights add up in
// it. Scores, weights and sums are fp32, each key's sum in one order.
//
// Bound: HBM, K is read once; near it the instructions (an exponential per score and, in 4
// bits, a conversion per two values). Single tokens, B=16 H=32/8 D=128, up to 8192 keys of 4
// bits (43 MB): 12 us, of which 3.5 pass before a wave has its first keys. B=2 H=32/8 N=32,
// 16384 keys of 16 bits (69 MB): 27 us, two blocks to a wave, each loaded in 4 us and
// multiplied in 8.
#include <climits>

#include "fa_paged.h"

namespace fa {
namespace {

// PER: workgroups of a CU.
template <int DIM, bool BF, int PER>
struct Weigh {
  static constexpr int kD = DIM, kTiles = 1, kRows = 16, kKeys = 64;
  static constexpr bool kBF = BF;
  static constexpr int kWaves = 4, kThreads = 64 * kWaves;
  static constexpr int kLine = INT_MAX;  // (an item's begin costs no more than a block's: no lead)
  static constexpr int kGrid = kCUs * PER;
  static constexpr float kPUnit = 1.f, kPRescale = 0.f;
};

// (a.window is 0 where every key is written; `window` hides keys from rows)
struct WeighArgs : PagedKernelArgs {
  const uint8_t* k_scale;
  long long scale_page, scale_head, scale_row;
  float* weights;
  long long weight_page, weight_head, weight_row;
  float scale;
  int hide_window;
  bool restart;
};

template <bool BF>
__device__ __forceinline__ floatx4 mfma4(half8 a, half8 b, floatx4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// FOUR: K is in 4 bits (its values are bf16, and q two bf16 numbers where it is fp16).
// FULL: the head dim is the width. ONE: all rows of a kv head are one tile: it stays in
// registers while the blocks go by, each loaded while the one before is multiplied. Else a
// block stays, as operands, and the tiles go by the same way. FEW: the rows of ONE are four
// at most, and stand in the tile four times, so that each quarter of the wave has a key
// tile's scores for itself (B=16 H=32/8 N=1, up to 8192 keys of 4 bits: 12 us instead of 15).
template <int D, bool FOUR, bool ONE, bool FEW>
constexpr int kPerCu = D <= 64 ? 3 + FEW : D <= 128 ? 2 + (ONE && FOUR) : 1 + (ONE && FOUR);
template <int D, bool BF, bool FOUR, bool FULL, bool ONE, bool FEW>
__global__ __launch_bounds__(256, (kPerCu<D, FOUR, ONE, FEW>)) void weights_kernel(const WeighArgs a) {
  static_assert(ONE || !FEW, "");
  using T = Weigh<D, BF, kPerCu<D, FOUR, ONE, FEW>>;
  constexpr int kWaves = T::kWaves, kChunks = D / 32, kQ = FOUR && !BF ? 2 : 1;
  // Operands' rows lie a row to a lane, whose loads would not join: they are loaded by
  // kLanes neighbouring lanes to a row, 16 bytes each, and go through LDS, where a row is
  // an odd number of 16 bytes (their banks differ). At B=2 H=32/8 N=32 D=128, 16384 keys in
  // 16 bits: 27 us instead of 32, and 3.9 M of L1's accesses instead of 13.7 M.
  constexpr int kUnits = FOUR ? D / 32 : D / 8, kLoads = (kUnits + 3) / 4;  // of a row
  constexpr int kLanes = kUnits < 3 ? kUnits : 4, kRowsAtOnce = 64 / kLanes;
  constexpr int kStride = kUnits | 1, kQStride = (D / 8) | 1;
  constexpr int kStage = (FOUR ? 64 : 16) * kStride;
  __shared__ u32x4 lds[kWaves][kStage + (ONE ? 0 : 16 * kQStride)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  u32x4 *const stage = lds[wave], *const q_stage = lds[wave] + kStage;
  const int wg = xcd_work_index(T::kGrid);
  const int l16 = lane & 15, g = lane >> 4;
  Line<T> line(a, lane);
  const int wg0 = wg * line.stretch, wg1 = min(wg0 + line.stretch, line.total);
  if (wg0 >= wg1) return;
  const bool single = line.stretch < kWaves;
  int pos = min(wg0 + (single ? wave : wave * line.stretch / kWaves), wg1);
  const int end = min(wg0 + (single ? wave + 1 : (wave + 1) * line.stretch / kWaves), wg1);
  if (pos >= end) return;
  int b, start;
  line.locate(pos, b, start);
  Keys<T> keys = line.keys(b);
  int item = (pos - start) / line.units(keys);
  start += item * line.units(keys);
  constexpr int kUnit = FOUR ? 1 : 2;
  const int page_mask = (1 << a.page_shift) - 1, dr = FULL ? D : a.dr;
  const int rows = a.group * a.N, row_tiles = (rows + 15) / 16;
  const float over_n = __builtin_amdgcn_rcpf((float)a.N);
  // Row r of a kv head as query head and row of it. (r < 2^24: off by one at most.)
  auto split = [&](int r, int& head, int& n) {
    head = (int)(((float)r + 0.5f) * over_n);
    n = r - head * a.N;
    if (n < 0) {
      --head;
      n += a.N;
    } else if (n >= a.N) {
      ++head;
      n -= a.N;
    }
  };

  // Where a lane's operand i of q begins.
  auto q_dim = [&](int i) { return FOUR ? D / 4 * g + 8 * i : 32 * i + 8 * g; };
  // (16 rows on: hop_n of them in a head, or into the next.)
  const int hop_n = 16 % a.N;
  const long long hop = 16 / a.N * (long long)a.stq.h + hop_n * (long long)a.stq.n;
  const long long hop_next = hop + a.stq.h - a.N * (long long)a.stq.n;

  while (pos < end) {
    const int units = line.units(keys), from = pos - start, upto = min(from + end - pos, units);
    const int hkv = item;
    const int j0 = keys.first + max(from - line.lead, 0);
    const int j1 = keys.len > keys.lo ? keys.first + max(upto - line.lead, 0) : j0;
    const int* table = a.table + b * a.table_stride;
    const int last_page = max(keys.len - 1, 0) >> a.page_shift;
    const uint8_t* base_k = (const uint8_t*)a.k + kUnit * hkv * a.head_stride;
    const uint8_t* base_s = FOUR ? a.k_scale + hkv * a.scale_head : nullptr;
    float* base_w = a.weights + hkv * a.weight_head;
    const float* lse_rows = a.lse + ((size_t)b * a.Hq + hkv * a.group) * a.N;
    int p0 = 0, held = 0;  // pages p0 .. p0 + 63 of the request are in the lanes
    auto fetch = [&](int j) {
      p0 = max(j * 64, keys.lo) >> a.page_shift;
      held = table[min(p0 + lane, last_page)];
      asm volatile("" : "+v"(held));  // (waited for here: behind a branch all loads would be)
    };

    // A block as it is loaded: K's rows, the words that hold the scales of key `lane`, from
    // byte `sub` of the first on, and the weight of that key.
    constexpr int kWords = D > 128 ? 3 : 2;
    struct Block {
      u32x4 rows[64 / kRowsAtOnce][kLoads];
      uint32_t words[FOUR ? kWords : 1], sub;
      float before;
      float* at;  // null where the lane has no key of the request
      bool fresh;
    };
    // (strides are below 2^31)
    auto place = [](int page, long long page_stride, int row, long long row_stride) {
      return (uint64_t)(uint32_t)page * (uint32_t)page_stride +
             (uint64_t)(uint32_t)row * (uint32_t)row_stride;
    };
    typedef __attribute__((address_space(1))) const uint32_t Word;
    auto load = [&](Block& x, int j) {
      if ((min(j * 64 + 64, keys.len) - 1) >> a.page_shift > p0 + 63) fetch(j);
      const int key = min(max(j * 64 + lane, keys.lo), keys.len - 1);
      const int page = __shfl(held, (key >> a.page_shift) - p0);
      const bool there = page >= 0 && page < a.pages;
      const int row = key & page_mask, my_page = there ? page : 0;
      x.at = there && key == j * 64 + lane ? base_w + place(page, a.weight_page, row, a.weight_row)
                                           : nullptr;
      x.fresh = a.restart || key >= keys.len - a.N;
      x.before = x.at && !x.fresh ? *x.at : 0.f;
      if constexpr (FOUR) {
        // (words that hold a scale of the row: none lies behind the pool)
        const uint64_t first = (uint64_t)base_s + place(my_page, a.scale_page, row, a.scale_row);
        const uint64_t from = first & ~3ull, upto = (first + dr / 32 - 1) & ~3ull;
        x.sub = (uint32_t)first & 3;
        x.words[0] = *(Word*)from;
        if constexpr (kWords == 3) x.words[1] = *(Word*)(from + 4 < upto ? from + 4 : upto);
        x.words[kWords - 1] = *(Word*)upto;
      }
      const uint64_t k_at = kUnit * place(my_page, a.page_stride, row, a.row_stride);
#pragma unroll
      for (int t = 0; t < 64 / kRowsAtOnce; ++t) {
        const int i = t * kRowsAtOnce + lane / kLanes;
        const uint32_t low = __shfl((uint32_t)k_at, i), high = __shfl((uint32_t)(k_at >> 32), i);
        const uint8_t* k = base_k + ((uint64_t)high << 32 | low);
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          const int unit = min(4 * e + lane % kLanes, kUnits - 1);
          const bool is = FULL || (FOUR ? 32 : 8) * unit < dr;
          // (behind the head dim the first unit again: finite values that meet zeros of q)
          if constexpr (FOUR)
            x.rows[t][e] = *reinterpret_cast<const u32x4*>(k + 16 * (is ? unit : 0));
          else
            x.rows[t][e] = load16(reinterpret_cast<const half_t*>(k) + 8 * unit, is);
        }
      }
    };
    auto put = [&](u32x4* to, int stride, int row, int e, u32x4 x) {
      const int unit = 4 * e + lane % kLanes;
      if (kUnits % kLanes == 0 || unit < kUnits) to[row * stride + unit] = x;
    };
    // Its operands: first all of it (in 4 bits), then a tile at a time.
    auto begin_operands = [&](const Block& x) {
      if constexpr (FOUR)
#pragma unroll
        for (int t = 0; t < 64 / kRowsAtOnce; ++t)
#pragma unroll
          for (int e = 0; e < kLoads; ++e)
            put(stage, kStride, t * kRowsAtOnce + lane / kLanes, e, x.rows[t][e]);
    };
    auto operands = [&](const Block& x, int t, half8 (&k)[kChunks]) {
      if constexpr (FOUR) {
        // The scales of the row, then of the lane's quarter of it (of either half where it is
        // 64 values; in 96 a quarter ends in the next scale's).
        uint32_t word = __builtin_amdgcn_alignbit(x.words[1], x.words[0], 8 * x.sub);
        word = __shfl(word, 16 * t + l16);
        if constexpr (kWords == 3) {
          const uint32_t high = __builtin_amdgcn_alignbit(x.words[2], x.words[1], 8 * x.sub);
          const uint32_t second = __shfl(high, 16 * t + l16);
          word = g < 2 ? word : second;
        }
        float two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int block = D == 256  ? 2 * (g & 1) + i
                            : D == 96 ? (3 * g + 2 * i) / 4
                                      : kChunks * g / 4;
          two[i] = __uint_as_float(__builtin_amdgcn_alignbit(word, word, (8 * block + 9u) & 31u));
          if constexpr (!FULL) two[i] = 64 * g + 32 * i < dr ? two[i] : 1.f;
        }
        uint32_t codes[kChunks];
        const char* const quarter = (const char*)(stage + (16 * t + l16) * kStride) + 4 * kChunks * g;
        __builtin_memcpy(codes, __builtin_assume_aligned(quarter, 4), 4 * kChunks);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const float scale = D == 96 ? (i == 0 || (i == 1 && g != 1) ? two[0] : two[1])
                                      : two[D == 256 ? i / 4 : 0];
          const uint32_t c = codes[i];
          k[i] = as_half8(u32x4{
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3))});
        }
      } else {
#pragma unroll
        for (int e = 0; e < kLoads; ++e) put(stage, kStride, lane / kLanes, e, x.rows[t][e]);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) k[i] = as_half8(stage[l16 * kStride + 4 * i + g]);
      }
    };
    // A tile of rows: q, of row lane % 16 (ONE) or as it goes to LDS, and lse of the rows that
    // the lane has scores of, 4 row_group .. 4 row_group + 3. They go by from the first tile
    // to the last, and again; lanes behind the last row keep the row they had.
    struct Rows {
      u32x4 q[kChunks];
      float lse[4];
    };
    const int row_group = FEW ? 0 : g;
    const auto lse_rsrc = make_rsrc(lse_rows, 4u * rows);
    const int my_row = FEW ? lane % 4 : ONE ? l16 : lane / 4;
    const half_t* q0;
    int n0;
    {
      int head;
      split(min(my_row, rows - 1), head, n0);
      q0 = a.q + b * a.stq.b + (hkv * a.group + head) * a.stq.h + n0 * (long long)a.stq.n;
    }
    const half_t* q_at = q0;
    int n_at = n0;
    auto load_rows = [&](Rows& x, int rt) {
      if (rt == 0) {
        q_at = q0;
        n_at = n0;
      } else if (16 * rt + my_row < rows) {
        n_at += hop_n;
        q_at += n_at >= a.N ? hop_next : hop;
        n_at -= n_at >= a.N ? a.N : 0;
      }
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int d = ONE ? q_dim(i) : 32 * i + 8 * (lane % 4);
        x.q[i] = load16(q_at + d, FULL || d < dr);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        x.lse[r] = buf_load_f32(lse_rsrc, 64 * rt + 16 * row_group + 4 * r, 0);
    };
    // Its operands.
    auto split_q = [&](const Rows& x, half8 (&q)[kQ][kChunks]) {
      if constexpr (!ONE)
#pragma unroll
        for (int i = 0; i < kChunks; ++i) q_stage[lane / 4 * kQStride + 4 * i + lane % 4] = x.q[i];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const half8 both = as_half8(ONE ? x.q[i] : q_stage[l16 * kQStride + q_dim(i) / 8]);
        q[0][i] = both;
        if constexpr (kQ == 2) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = (float)both[e];
            q[0][i][e] = to16<true>(f);
            const float rest = f - from16<true>(q[0][i][e]);
            q[kQ - 1][i][e] = to16<true>(__builtin_isfinite(f) ? rest : 0.f);
          }
        }
      }
    };
    const int all_lo = a.hide_window > 0 ? max(0, keys.len - a.hide_window) : 0;
    const int all_hi = a.causal ? keys.len - a.N + 1 : keys.len;
    // What rows score above their lse with the block's keys (tile t, or the lane's own); operands(t,
    // k): those of key tile t.
    constexpr int kOwn = FEW ? 1 : 4;
    auto scores = [&](const Rows& x, const half8 (&q)[kQ][kChunks], floatx4 (&z)[kOwn],
                      auto&& operands) {
      floatx4 s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        half8 k[kChunks];
        operands(t, k);
        s[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < kQ; ++y)
#pragma unroll
          for (int i = 0; i < kChunks; ++i) s[t] = mfma4<BF || FOUR>(q[y][i], k[i], s[t]);
      }
      // (score - lse first: exact near 0, where the weights are large)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (FEW) s[0][r] = g < 2 ? (g == 0 ? s[0][r] : s[1][r]) : g == 2 ? s[2][r] : s[3][r];
#pragma unroll
        for (int t = 0; t < kOwn; ++t) z[t][r] = fmaf(s[t][r], a.scale, -x.lse[r]);
      }
    };
    // Adds to acc the weights that they, of tile rt, give the keys.
    auto weigh = [&](floatx4 (&z)[kOwn], int rt, int j, float (&acc)[kOwn]) {
      if (j * 64 < all_lo || j * 64 + 64 > all_hi || a.alibi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int head, n;
          split(min(16 * rt + 4 * row_group + r, rows - 1), head, n);
          const int at = keys.len - a.N + n;
          const float slope = a.alibi ? a.alibi[hkv * a.group + head] : 0.f;
          const int lo = a.hide_window > 0 ? max(0, at - a.hide_window + 1) : 0;
          const int hi = a.causal ? min(keys.len, at + 1) : keys.len;
#pragma unroll
          for (int t = 0; t < kOwn; ++t) {
            const int key = j * 64 + (FEW ? lane : 16 * t + l16);
            const float biased = fmaf(-slope, (float)abs(at - key), z[t][r]);
            z[t][r] = key < lo || key >= hi ? -INFINITY : a.alibi ? biased : z[t][r];
          }
        }
      }
      if (16 * rt + (FEW ? 4 : 16) > rows)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < kOwn; ++t)
            z[t][r] = 16 * rt + 4 * row_group + r < rows ? z[t][r] : -INFINITY;
#pragma unroll
      for (int t = 0; t < kOwn; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t] += fast_exp2(z[t][r] * kLog2e);
    };
    auto store = [&](float* at, float before, const float (&acc)[kOwn]) {
      float sum = acc[0];
      if constexpr (!FEW)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          float y = acc[t] + __shfl_xor(acc[t], 16);
          y += xor32(y);
          sum = g == t ? y : sum;
        }
      if (at) *at = before + sum;
    };

    if (j0 < j1) {
      fetch(j0);
      if constexpr (ONE) {
        Rows now;
        load_rows(now, 0);
        half8 q[kQ][kChunks];
        Block x;
        load(x, j0);
        split_q(now, q);
        for (int j = j0; j < j1; ++j) {
          // (behind the last block that block again: a branch around the loads would have all
          // of them waited for)
          Block next;
          if constexpr (FOUR) load(next, min(j + 1, j1 - 1));
          float acc[kOwn] = {};
          floatx4 z[kOwn];
          begin_operands(x);
          scores(now, q, z, [&](int t, half8 (&k)[kChunks]) { operands(x, t, k); });
          weigh(z, 0, j, acc);
          float* const at = x.at;
          const float before = x.before;
          // (the next block is waited for ahead of the store, which it would wait for too)
          if constexpr (FOUR)
            x = next;
          else if (j + 1 < j1)
            load(x, j + 1);
          store(at, before, acc);
        }
      } else {
        // Two tiles of rows by turns: one is loaded while the other is multiplied, the first
        // again for the next block. (The next block's keys are not: what the rows wait for
        // would wait for those too, 31 us instead of 27.)
        Rows even, odd;
        load_rows(even, 0);
        for (int j = j0; j < j1; ++j) {
          Block x;
          load(x, j);
          begin_operands(x);
          half8 k[4][kChunks];
#pragma unroll
          for (int t = 0; t < 4; ++t) operands(x, t, k[t]);
          float acc[kOwn] = {};
          auto tile = [&](const Rows& rows, int rt) {
            half8 q[kQ][kChunks];
            split_q(rows, q);
            floatx4 z[kOwn];
            scores(rows, q, z, [&](int t, half8 (&tile)[kChunks]) {
#pragma unroll
              for (int i = 0; i < kChunks; ++i) tile[i] = k[t][i];
            });
            weigh(z, rt, j, acc);
          };
          for (int rt = 0; rt < row_tiles; rt += 2) {
            load_rows(odd, rt + 1);
            tile(even, rt);
            load_rows(even, rt + 2 < row_tiles ? rt + 2 : 0);
            if (rt + 1 < row_tiles) tile(odd, rt + 1);
          }
          store(x.at, x.before, acc);
        }
      }
    }
    pos += upto - from;
    start += units;
    if (++item == a.items && pos < end) {
      if (++b == a.B) break;
      item = 0;
      keys = line.keys(b);
    }
  }
}

}  // namespace

template <>
hipError_t launch_paged_weights_w<FA_WIDTH, FA_BF>(const PagedArgs& a, const KeyWeights& w,
                                                   bool restart) {
  WeighArgs d{};
  paged_args<Weigh<FA_WIDTH, FA_BF, 1>>(d, a);
  d.n_groups = 1;
  d.items = a.Hkv;
  d.k_scale = a.scales.k;
  d.scale_page = a.scales.page_stride;
  d.scale_head = a.scales.head_stride;
  d.scale_row = a.scales.row_stride;
  d.weights = w.w;
  d.weight_page = w.page_stride;
  d.weight_head = w.head_stride;
  d.weight_row = w.row_stride;
  d.scale = a.scale > 0.f ? a.scale : 1.f / sqrtf((float)a.D);
  d.hide_window = d.window;
  if (restart) d.window = 0;
  d.restart = restart;
  auto launch = [&](auto four, auto full, auto one, auto few) {
    constexpr bool kFour = decltype(four)::value, kFull = decltype(full)::value;
    constexpr bool kOne = decltype(one)::value, kFew = decltype(few)::value;
    using T = Weigh<FA_WIDTH, FA_BF, kPerCu<FA_WIDTH, kFour, kOne, kFew>>;
    hipLaunchKernelGGL((weights_kernel<FA_WIDTH, FA_BF, kFour, kFull, kOne, kFew>), dim3(T::kGrid),
                       dim3(T::kThreads), 0, (hipStream_t)a.stream, d);
    return hipGetLastError();
  };
  using std::false_type, std::true_type;
  auto by_rows = [&](auto four, auto full) {
    if (d.group * d.N <= 4) return launch(four, full, true_type{}, true_type{});
    return d.group * d.N <= 16 ? launch(four, full, true_type{}, false_type{})
                               : launch(four, full, false_type{}, false_type{});
  };
  // (4-bit rows are whole blocks of 32: of the widths, 256 alone serves narrower ones)
  const bool full = a.D == FA_WIDTH;
  using Narrow4 = std::integral_constant<bool, FA_WIDTH != 256>;
  if (a.scales.k) return full ? by_rows(true_type{}, true_type{}) : by_rows(true_type{}, Narrow4{});
  return full ? by_rows(false_type{}, true_type{}) : by_rows(false_type{}, false_type{});
}

}  // namespace fa
