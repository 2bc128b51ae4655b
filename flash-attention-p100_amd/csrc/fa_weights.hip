// The weight that each key of a paged cache gets from the newest rows of its request,
// given the rows' lse: w[key, kv head] += sum over the rows that see the key and the
// query heads of the group of exp(score - lse). (What eviction by accumulated attention
// goes by: fa_evict.hip.) No counterpart in the reference, which has no cache.
//
// Bound: HBM, K is read once, a quarter or less of the bytes that attention needs in
// 16 bits where few rows share a key. The lse is known, so keys do not depend on each
// other: the blocks of 64 keys of all requests and kv heads lie on one line that the
// waves divide evenly (as in fa_paged.hip), a wave holds a block of K as operands and
// goes over all rows of the kv head, 16 at a time, on v_mfma_f32_16x16x32, S = Q K^T: a
// lane has one key of a tile, so the rows' weights add up in it. Scores, weights and
// sums are fp32, each key's sum in one order.
#include "fa_paged.h"

namespace fa {
namespace {

// PER: workgroups of a CU.
template <int DIM, bool BF, int PER>
struct Weigh {
  static constexpr int kD = DIM, kTiles = 1, kRows = 16, kKeys = 64;
  static constexpr bool kBF = BF;
  static constexpr int kWaves = 4, kLine = kWaves, kThreads = 64 * kWaves;
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
// block stays, as operands, and the tiles go by the same way.
template <int D, bool FOUR, bool ONE>
constexpr int kPerCu = D <= 64 ? 3 : D <= 128 ? (ONE && FOUR ? 3 : 2) : ONE && FOUR ? 2 : 1;
template <int D, bool BF, bool FOUR, bool FULL, bool ONE>
__global__ __launch_bounds__(256, (kPerCu<D, FOUR, ONE>)) void weights_kernel(const WeighArgs a) {
  using T = Weigh<D, BF, kPerCu<D, FOUR, ONE>>;
  constexpr int kWaves = T::kWaves, kChunks = D / 32, kQ = FOUR && !BF ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
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
    };

    // A block as it is loaded: K's rows (of key 16 t + lane % 16 in 16 bits the chunks 4 i + g,
    // in 4 a quarter of the row and the words of its scales), and the weight of key `lane`.
    constexpr int kScales = D == 96 || D == 256 ? 2 : 1;
    struct Block {
      u32x4 rows[FOUR ? 1 : 4][FOUR ? 1 : kChunks];
      uint32_t codes[FOUR ? 4 : 1][kChunks], scale[4][kScales], bit[4][kScales];
      float before;
      float* at;  // null where the lane has no key of the request
      bool fresh;
    };
    auto load = [&](Block& x, int j) {
      if ((min(j * 64 + 64, keys.len) - 1) >> a.page_shift > p0 + 63) fetch(j);
      const int key = min(max(j * 64 + lane, keys.lo), keys.len - 1);
      const int page = __shfl(held, (key >> a.page_shift) - p0);
      const bool there = page >= 0 && page < a.pages;
      const int row = key & page_mask;
      x.at = there && key == j * 64 + lane ? base_w + (there ? page : 0) * a.weight_page + row * a.weight_row : nullptr;
      x.fresh = a.restart || key >= keys.len - a.N;
      x.before = x.at && !x.fresh ? *x.at : 0.f;
      const int my_page = there ? page : 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int p = __shfl(my_page, 16 * t + l16), r = __shfl(row, 16 * t + l16);
        const uint8_t* k = base_k + kUnit * (p * a.page_stride + r * a.row_stride);
        if constexpr (FOUR) {
          const uint8_t* scales = base_s + p * a.scale_page + r * a.scale_row;
          const bool begins = FULL || 64 * g < dr, both = FULL || 64 * g + 32 < dr;
          const uint8_t* q = k + 4 * kChunks * (begins ? g : 0);
          if constexpr (kChunks < 4) {
            __builtin_memcpy(x.codes[t], __builtin_assume_aligned(q, 4), 4 * kChunks);
          } else {
#pragma unroll
            for (int h = 0; h < kChunks / 4; ++h) {
              const u32x4 v = *reinterpret_cast<const u32x4*>(q + (both ? 16 * h : 0));
#pragma unroll
              for (int i = 0; i < 4; ++i) x.codes[t][4 * h + i] = v[i];
            }
          }
#pragma unroll
          for (int i = 0; i < kScales; ++i) {
            const int block = !begins ? 0 : D == 256 ? 2 * g + (both ? i : 0) : (kChunks * g + 2 * i) / 4;
            const uint8_t* s = scales + block;
            const uint32_t sub = (uint32_t)((uintptr_t)s & 3);
            x.bit[t][i] = 8 * sub;
            x.scale[t][i] = *reinterpret_cast<const uint32_t*>(s - sub);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kChunks; ++i)
            x.rows[t][i] = load16(reinterpret_cast<const half_t*>(k) + 32 * i + 8 * g, FULL || 32 * i + 8 * g < dr);
        }
      }
    };
    // Its operands, a tile at a time (values past the head dim meet zeros of q: finite ones).
    auto operands = [&](const Block& x, int t, half8 (&k)[kChunks]) {
      if constexpr (FOUR) {
        float two[2];
#pragma unroll
        for (int i = 0; i < kScales; ++i)
          two[i] = __uint_as_float(__builtin_amdgcn_alignbit(x.scale[t][i], x.scale[t][i], (x.bit[t][i] + 9u) & 31u));
        if constexpr (kScales == 1) two[1] = two[0];
        if constexpr (!FULL) {
          two[0] = 64 * g < dr ? two[0] : 1.f;
          two[1] = 64 * g + 32 < dr ? two[1] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const float scale = D == 96 ? (i == 0 || (i == 1 && g != 1) ? two[0] : two[1]) : two[D == 256 ? i / 4 : 0];
          const uint32_t c = x.codes[t][i];
          k[i] = as_half8(u32x4{
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3))});
        }
      } else {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) k[i] = as_half8(x.rows[t][i]);
      }
    };
    // A tile of rows: q of row lane % 16, lse of rows 4 g .. 4 g + 3 (+inf, a weight of 0,
    // where there is none).
    struct Rows {
      half8 q[kChunks];
      float lse[4];
    };
    auto load_rows = [&](Rows& x, int rt) {
      int head, n;
      split(min(16 * rt + l16, rows - 1), head, n);
      const half_t* q = a.q + b * a.stq.b + (hkv * a.group + head) * a.stq.h + (size_t)n * a.stq.n;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int d = FOUR ? D / 4 * g + 8 * i : 32 * i + 8 * g;
        x.q[i] = as_half8(load16(q + d, FULL || d < dr));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x.lse[r] = lse_rows[min(16 * rt + 4 * g + r, rows - 1)];
    };
    const int all_lo = a.hide_window > 0 ? max(0, keys.len - a.hide_window) : 0;
    const int all_hi = a.causal ? keys.len - a.N + 1 : keys.len;
    // Adds to acc the weights that rows of tile rt give the keys of tile t.
    auto weigh = [&](const Rows& x, const half8 (&q)[kQ][kChunks], const half8 (&k)[kChunks], int rt, int j, int t,
                     float& acc) {
      floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < kQ; ++y)
#pragma unroll
        for (int i = 0; i < kChunks; ++i) s = mfma4<BF || FOUR>(q[y][i], k[i], s);
      const int key = j * 64 + 16 * t + l16;
      const bool edge = j * 64 < all_lo || j * 64 + 64 > all_hi || 16 * rt + 16 > rows;
      // (score - lse first: exact near 0, where the weights are large)
      float z[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) z[r] = fmaf(s[r], a.scale, -x.lse[r]);
      if (edge || a.alibi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * rt + 4 * g + r;
          int head, n;
          split(min(row, rows - 1), head, n);
          const int at = keys.len - a.N + n;
          if (a.alibi) z[r] = fmaf(-a.alibi[hkv * a.group + head], (float)abs(at - key), z[r]);
          const int lo = a.hide_window > 0 ? max(0, at - a.hide_window + 1) : 0;
          const int hi = row >= rows ? 0 : a.causal ? min(keys.len, at + 1) : keys.len;
          if (key < lo || key >= hi) z[r] = -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) acc += fast_exp2(z[r] * kLog2e);
    };
    auto split_q = [&](const Rows& x, half8 (&q)[kQ][kChunks]) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        q[0][i] = x.q[i];
        if constexpr (kQ == 2) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = (float)x.q[i][e];
            q[0][i][e] = to16<true>(f);
            const float rest = f - from16<true>(q[0][i][e]);
            q[kQ - 1][i][e] = to16<true>(__builtin_isfinite(f) ? rest : 0.f);
          }
        }
      }
    };
    auto store = [&](const Block& x, const float (&acc)[4]) {
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float y = acc[t] + __shfl_xor(acc[t], 16);
        y += xor32(y);
        sum = g == t ? y : sum;
      }
      if (x.at) *x.at = x.before + sum;
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
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            half8 k[kChunks];
            operands(x, t, k);
            weigh(now, q, k, 0, j, t, acc[t]);
          }
          if constexpr (FOUR) {
            store(x, acc);
            x = next;
          } else {
            const Block old = x;
            if (j + 1 < j1) load(x, j + 1);
            store(old, acc);
          }
        }
      } else {
        for (int j = j0; j < j1; ++j) {
          Block x;
          Rows now, next;
          load(x, j);
          load_rows(now, 0);
          half8 k[4][kChunks];
#pragma unroll
          for (int t = 0; t < 4; ++t) operands(x, t, k[t]);
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          for (int rt = 0; rt < row_tiles; ++rt) {
            load_rows(next, min(rt + 1, row_tiles - 1));
            half8 q[kQ][kChunks];
            split_q(now, q);
#pragma unroll
            for (int t = 0; t < 4; ++t) weigh(now, q, k[t], rt, j, t, acc[t]);
            now = next;
          }
          store(x, acc);
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
hipError_t launch_paged_weights_w<FA_WIDTH, FA_BF>(const PagedArgs& a, const KeyWeights& w, bool restart) {
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
  auto launch = [&](auto four, auto full, auto one) {
    constexpr bool kFour = decltype(four)::value, kFull = decltype(full)::value, kOne = decltype(one)::value;
    using T = Weigh<FA_WIDTH, FA_BF, kPerCu<FA_WIDTH, kFour, kOne>>;
    hipLaunchKernelGGL((weights_kernel<FA_WIDTH, FA_BF, kFour, kFull, kOne>), dim3(T::kGrid), dim3(T::kThreads), 0,
                       (hipStream_t)a.stream, d);
    return hipGetLastError();
  };
  using std::false_type, std::true_type;
  auto by_rows = [&](auto four, auto full) {
    return d.group * d.N <= 16 ? launch(four, full, true_type{}) : launch(four, full, false_type{});
  };
  // (4-bit rows are whole blocks of 32: of the widths, 256 alone serves narrower ones)
  const bool full = a.D == FA_WIDTH;
  using Narrow4 = std::integral_constant<bool, FA_WIDTH != 256>;
  if (a.scales.k) return full ? by_rows(true_type{}, true_type{}) : by_rows(true_type{}, Narrow4{});
  return full ? by_rows(false_type{}, true_type{}) : by_rows(false_type{}, false_type{});
}

}  // namespace fa
