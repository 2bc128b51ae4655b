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

template <int DIM, bool BF>
struct Weigh {
  static constexpr int kD = DIM, kTiles = 1, kRows = 16, kKeys = 64;
  static constexpr bool kBF = BF;
  static constexpr int kWaves = 4, kLine = kWaves, kThreads = 64 * kWaves;
  static constexpr int kGrid = kCUs * (DIM > 128 ? 2 : 4);
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
// FULL: the head dim is the width.
template <int D, bool BF, bool FOUR, bool FULL>
__global__ __launch_bounds__(256) void weights_kernel(const WeighArgs a) {
  using T = Weigh<D, BF>;
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
  const int unit = FOUR ? 1 : 2;
  const int page_mask = (1 << a.page_shift) - 1, dr = FULL ? D : a.dr;
  const int rows = a.group * a.N, row_tiles = (rows + 15) / 16;

  while (pos < end) {
    const int units = line.units(keys), from = pos - start, upto = min(from + end - pos, units);
    const int hkv = item;
    const int j0 = keys.first + max(from - line.lead, 0);
    const int j1 = keys.len > keys.lo ? keys.first + max(upto - line.lead, 0) : j0;
    const int* table = a.table + b * a.table_stride;
    const uint8_t* base_k = (const uint8_t*)a.k + unit * hkv * a.head_stride;
    const uint8_t* base_s = FOUR ? a.k_scale + hkv * a.scale_head : nullptr;
    float* base_w = a.weights + hkv * a.weight_head;
    for (int j = j0; j < j1; ++j) {
      // A lane's own key (its page, its weight), and those of the tiles.
      const int my_key = min(max(j * 64 + lane, keys.lo), keys.len - 1);
      int my_page = table[my_key >> a.page_shift];
      const bool ok = my_page >= 0 && my_page < a.pages;
      my_page = ok ? my_page : 0;
      float* const my_w = base_w + my_page * a.weight_page + (my_key & page_mask) * a.weight_row;
      const bool mine = ok && j * 64 + lane == my_key;
      const bool fresh = a.restart || my_key >= keys.len - a.N;
      const float before = mine && !fresh ? *my_w : 0.f;
      half8 k[4][kChunks];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int page = __shfl(my_page, 16 * t + l16), key = __shfl(my_key, 16 * t + l16);
        const uint8_t* row = base_k + unit * (page * a.page_stride + (key & page_mask) * a.row_stride);
        if constexpr (FOUR) {
          const uint8_t* scales = base_s + page * a.scale_page + (key & page_mask) * a.scale_row;
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int d = D / 4 * g + 8 * i;  // (of a quarter of the row)
            const bool there = FULL || d < dr;
            const uint32_t codes = there ? *reinterpret_cast<const uint32_t*>(row + d / 2) : 0u;
            const float scale = __uint_as_float((there ? (uint32_t)scales[d / 32] : 127u) << 23);
            auto two = [&](auto sel) {
              return __builtin_bit_cast(
                  uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, decltype(sel)::value));
            };
            k[t][i] = as_half8(u32x4{two(std::integral_constant<int, 0>{}), two(std::integral_constant<int, 1>{}),
                                     two(std::integral_constant<int, 2>{}), two(std::integral_constant<int, 3>{})});
          }
        } else {
#pragma unroll
          for (int i = 0; i < kChunks; ++i)
            k[t][i] = as_half8(load16(reinterpret_cast<const half_t*>(row) + 32 * i + 8 * g,
                                      FULL || 32 * i + 8 * g < dr));
        }
      }
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int rt = 0; rt < row_tiles; ++rt) {
        half8 q[kQ][kChunks];
        const Row<16> mine(a, hkv, rt, l16);
        const half_t* qrow = a.q + b * a.stq.b + mine.hq * a.stq.h + (size_t)mine.n * a.stq.n;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const int d = FOUR ? D / 4 * g + 8 * i : 32 * i + 8 * g;
          const half8 x = as_half8(load16(qrow + d, FULL || d < dr));
          if constexpr (kQ == 1) {
            q[0][i] = x;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float f = (float)x[e];
              q[0][i][e] = to16<true>(f);
              const float rest = f - from16<true>(q[0][i][e]);
              q[kQ - 1][i][e] = to16<true>(__builtin_isfinite(f) ? rest : 0.f);
            }
          }
        }
        // The four rows of this lane's scores.
        float lse[4], slope[4];
        int lo[4], hi[4], at[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Row<16> row(a, hkv, rt, 4 * g + r);
          lse[r] = a.lse[((size_t)b * a.Hq + row.hq) * a.N + row.n];
          slope[r] = a.alibi ? a.alibi[row.hq] : 0.f;
          at[r] = keys.len - a.N + row.n;
          lo[r] = a.hide_window > 0 ? max(0, at[r] - a.hide_window + 1) : 0;
          hi[r] = !row.ok ? 0 : a.causal ? min(keys.len, at[r] + 1) : keys.len;
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = 0; x < kQ; ++x)
#pragma unroll
            for (int i = 0; i < kChunks; ++i) s = mfma4<BF || FOUR>(q[x][i], k[t][i], s);
          const int key = j * 64 + 16 * t + l16;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (score - lse first: exact near 0, where the weights are large)
            float z = fmaf(s[r], a.scale, -lse[r]);
            if (a.alibi) z = fmaf(-slope[r], (float)abs(at[r] - key), z);
            acc[t] += key >= lo[r] && key < hi[r] ? fast_exp2(z * kLog2e) : 0.f;
          }
        }
      }
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float x = acc[t] + __shfl_xor(acc[t], 16);
        x += xor32(x);
        sum = g == t ? x : sum;
      }
      if (mine) *my_w = before + sum;
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
  using T = Weigh<FA_WIDTH, FA_BF>;
  WeighArgs d{};
  paged_args<T>(d, a);
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
  // (4-bit rows are whole blocks of 32: of the widths, 256 alone serves narrower ones)
  constexpr bool kFull4 = FA_WIDTH != 256;
  const bool full = a.D == FA_WIDTH;
  const auto kernel = a.scales.k ? (full ? weights_kernel<FA_WIDTH, FA_BF, true, true>
                                         : weights_kernel<FA_WIDTH, FA_BF, true, kFull4>)
                                 : (full ? weights_kernel<FA_WIDTH, FA_BF, false, true>
                                         : weights_kernel<FA_WIDTH, FA_BF, false, false>);
  hipLaunchKernelGGL(kernel, dim3(T::kGrid), dim3(T::kThreads), 0, (hipStream_t)a.stream, d);
  return hipGetLastError();
}

}  // namespace fa
