// Attention of the newest tokens of each request over a paged cache in 4 bits. A row of
// K or V is codes of 4 bits (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) and a power
// of two per 32 of them, so a value is code * 2^(scale - 127). No counterpart in the
// reference, which has no cache.
//
// As in fa_paged.hip the key blocks of all requests lie on one line that the waves
// divide evenly, and the parts of an item meet in LDS and in paged_merge_kernel. A
// wave's step is a block of 64 keys for RT tiles of 16 query rows, on
// v_mfma_f32_16x16x32_bf16: S^T = K Q^T, then O^T += V^T P^T. Every value of the cache is
// exact in bf16 (a sign, two bits and an exponent), whatever q's format, and
// v_cvt_scalef32_pk_bf16_fp4 makes two of them from a byte, scale included:
//   * K: a lane's codes are an MFMA operand as they lie (key lane % 16, a quarter of the
//     row), so they go from memory to registers and need no LDS;
//   * V: the second product runs over keys, so the values are written to LDS as bf16 and
//     come back transposed (ds_read_b64_tr_b16).
// q in fp16 has 11 bits: two bf16 numbers, exactly, and two products. The probabilities
// are two bf16 numbers up to 32 rows (off by 2^-16), with more rows one, as in
// fa_paged.hip.
#include "fa_paged.h"

namespace fa {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int DIM, bool OUT_BF, int RT>
struct Paged4 {
  static constexpr int kD = DIM, kTiles = 1, kRowTiles = RT, kRows = 16 * RT, kKeys = 64;
  static constexpr bool kBF = OUT_BF;
  static constexpr int kWaves = DIM > 128 ? 4 : 8, kLine = kWaves, kThreads = 64 * kWaves;
  static constexpr int kGrid = kCUs;
  static constexpr float kPUnit = 1.f, kPRescale = kRescaleLog2;
  static constexpr int kBlocks = DIM / 32;  // of a row, each with its scale
  static constexpr int kQ = OUT_BF ? 1 : 2;  // bf16 operands of q
  static constexpr bool kTwoP = RT <= 2;
  // LDS rows of V: eight 16-byte chunks in a row of keys, two of each, lie in 16 bank
  // groups (the row's chunks are 2 more than a multiple of 4).
  static constexpr int kStride = 2 * DIM + 32;
  static constexpr int kTileBytes = kKeys * kStride;
  static constexpr int kFloats = 16 * DIM;  // a row tile's partial O
  static_assert(kFloats * 4 <= kTileBytes, "a part exceeds the wave's tile");
  __device__ __forceinline__ static bool joins(int stretch, int total, int items) {
    constexpr int kFrom = kLine < 4 ? kLine : 4;
    return stretch >= kFrom || (stretch >= 2 && total / 64 >= items);
  }
};

struct Paged4Args : PagedKernelArgs {
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  long long scale_page, scale_head, scale_row;
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
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// The maximum over lanes l, l ^ 16, l ^ 32 and l ^ 48, which hold the same query row.
__device__ __forceinline__ float max_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// FULL: the head dim is the width (else 160, 192 or 224 of 256).
template <class T, bool FULL>
__global__ __launch_bounds__(T::kThreads) void paged4_kernel(const Paged4Args a) {
  constexpr int D = T::kD, RT = T::kRowTiles, kWaves = T::kWaves, kLine = T::kLine;
  constexpr int kBlocks = T::kBlocks, kDwords = D / 32;  // of a row, and of a lane's quarter of it
  __shared__ __align__(1024) char vt[kWaves * T::kTileBytes];
  __shared__ float2 ml[kWaves * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  const int wg = xcd_work_index(T::kGrid);
  const int l16 = lane & 15, g = lane >> 4;
  Line<T> line(a, lane);
  if (wg == 0 && tid == 0) {
    a.sizes[0] = line.stretch;
    a.sizes[1] = line.total;
  }
  const int wg0 = wg * line.stretch, wg1 = min(wg0 + line.stretch, line.total);
  int4 owned = make_int4(0, 0, 0, 0);  // request, item, its start and units (none: 0)
  if (wg0 >= wg1) {
    if (lane == 0) a.owned[wg * kLine + wave] = owned;
    return;
  }
  const bool single = line.stretch < kLine;
  int pos = min(wg0 + (single ? wave : wave * line.stretch / kLine), wg1);
  const int end = min(wg0 + (single ? wave + 1 : (wave + 1) * line.stretch / kLine), wg1);
  int b, start;
  line.locate(min(pos, wg1 - 1), b, start);
  Keys<T> keys = line.keys(b);
  int item = (min(pos, wg1 - 1) - start) / line.units(keys);
  start += item * line.units(keys);  // of the item, from here on
  const bool joins = T::joins(line.stretch, line.total, a.B * a.items);
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
    int p0 = 0, held = 0;           // pages p0 .. p0 + 63 are in the lanes' `held`
    unsigned long long hidden = 0;  // of those, the ones outside the pool
    const uint8_t* base_k = (const uint8_t*)a.k + hkv * a.head_stride;
    const uint8_t* base_v = (const uint8_t*)a.v + hkv * a.head_stride;
    const uint8_t* base_ks = a.k_scale + hkv * a.scale_head;
    const uint8_t* base_vs = a.v_scale + hkv * a.scale_head;
    auto fetch = [&](int j) {  // pages for block j
      p0 = max(j * 64, keys.lo) >> a.page_shift;
      const int page = table[min(p0 + lane, last_page)];
      const bool ok = page >= 0 && page < a.pages;
      hidden = __ballot(!ok);
      held = ok ? page : 0;
    };
    auto place = [&](int j) {
      if ((min(j * 64 + 64, keys.len) - 1) >> a.page_shift > p0 + 63) fetch(j);
    };
    // Where key `x` of a block lies (rows outside the request's keys: one of its own).
    auto page_of = [&](int x, int& row) {
      const int key = min(max(x, keys.lo), keys.len - 1);
      row = key & page_mask;
      return (uint32_t)__shfl(held, (key >> a.page_shift) - p0);
    };
    // A block in registers: K's codes (key 16 t + lane % 16, a quarter of its row), V's
    // (unit u = lane + 64 i: block u % kBlocks of key u / kBlocks), and their scales.
    constexpr int kScales = D == 96 ? 3 : D == 256 ? 2 : 1;
    uint32_t kc[4][kDwords], ks[4][kScales], vs[kBlocks];
    u32x4 vc[kBlocks];
    auto load_k = [&](int j, bool live) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        int row;
        const uint32_t page = page_of(j * 64 + 16 * t + l16, row);
        const unsigned long long at = live ? (unsigned long long)page * page_bytes +
                                                 (unsigned long long)(uint32_t)row * row_bytes : 0;
        const unsigned long long sat = live ? (unsigned long long)page * scale_page +
                                                  (unsigned long long)(uint32_t)row * scale_row : 0;
        if constexpr (D == 256) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int blk = FULL || 64 * g + 32 * h < dr ? 2 * g + h : 0;
            const u32x4 x = *reinterpret_cast<const u32x4*>(base_k + at + 16 * blk);
            for (int i = 0; i < 4; ++i) kc[t][(4 * h + i) % kDwords] = x[i];
            ks[t][h % kScales] = FULL || 64 * g + 32 * h < dr ? base_ks[sat + blk] : 127u;
          }
        } else {
          __builtin_memcpy(kc[t], __builtin_assume_aligned(base_k + at + 4 * kDwords * g, kDwords == 3 ? 4 : 4 * kDwords),
                           4 * kDwords);
#pragma unroll
          for (int i = 0; i < kScales; ++i) ks[t][i] = base_ks[sat + (kDwords * g + i) / 4];
        }
      }
    };
    auto load_v = [&](int j, bool live) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int u = lane + 64 * i, key = u / kBlocks, blk = FULL || 32 * (u % kBlocks) < dr ? u % kBlocks : 0;
        int row;
        const uint32_t page = page_of(j * 64 + key, row);
        const unsigned long long at = live ? (unsigned long long)page * page_bytes +
                                                 (unsigned long long)(uint32_t)row * row_bytes : 0;
        const unsigned long long sat = live ? (unsigned long long)page * scale_page +
                                                  (unsigned long long)(uint32_t)row * scale_row : 0;
        vc[i] = *reinterpret_cast<const u32x4*>(base_v + at + 16 * blk);
        vs[i] = base_vs[sat + blk];
      }
    };

    if (j0 < j1) {
      fetch(j0);
      load_k(j0, true);
      load_v(j0, true);
    }
    LateArgs& qa = late_args();
    half8 q[RT][T::kQ][kDwords];
    float slope[RT], m_raw[RT], l[RT];
    int row_n[RT];
    floatx4 oacc[RT][D / 16];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const Row<T::kRows> row(qa, hkv, tile, 16 * rt + l16);
      const half_t* qrow = qa.q + b * qa.stq.b + row.hq * qa.stq.h + (size_t)row.n * qa.stq.n;
      row_n[rt] = row.n;
      slope[rt] = qa.alibi ? qa.alibi[row.hq] * qa.alibi_unit : 0.f;
      m_raw[rt] = -INFINITY;
      l[rt] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) oacc[rt][c] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kDwords; ++i) {
        const int d = D / 4 * g + 8 * i;
        const half8 x = as_half8(load16(qrow + d, FULL || d < dr));
        if constexpr (T::kBF) {
          q[rt][0][i] = x;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = (float)x[e];
            q[rt][0][i][e] = to16<true>(f);
            const float rest = f - from16<true>(q[rt][0][i][e]);
            q[rt][T::kQ - 1][i][e] = to16<true>(__builtin_isfinite(f) ? rest : 0.f);
          }
        }
      }
    }
    const int at0 = keys.len - qa.N, window = qa.window;
    const int all_lo = window > 0 ? max(0, keys.len - window) : 0;
    const int all_hi = qa.causal ? at0 + 1 : keys.len;
    const bool causal = qa.causal, biased = qa.alibi != nullptr;
    const float c = qa.scale_log2, thr_raw = qa.rescale;
    for (int j = j0; j < j1; ++j) {
      const unsigned long long hide = hidden;  // (of block j's pages, from page hide0 on)
      const int hide0 = p0;
      floatx4 s[RT][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kDwords; ++i) {
          // (a lane's quarter begins in block g kDwords / 4 and may end in another)
          const half8 k = values(kc[t][i], scale_of(ks[t][D == 256 ? i / 4 % kScales : i % kScales]));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int x = 0; x < T::kQ; ++x) s[rt][t] = mfma_bf16(k, q[rt][x][i], s[rt][t]);
        }
      }
      const bool more = j + 1 < j1;
      if (more) place(j + 1);
      load_k(more ? j + 1 : j, more);
      const int base = j * 64 + 4 * g;  // key of s[.][t][r]: base + 16 t + r
      const bool edge = j * 64 < all_lo || j * 64 + 64 > all_hi;
      half8 pb[RT][2], rest[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int at = at0 + row_n[rt];
        if (biased) {
          const float d0 = (float)(at - base);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[rt][e >> 2][e & 3] =
                fmaf(-slope[rt], fabsf(d0 - (float)(16 * (e >> 2) + (e & 3))), s[rt][e >> 2][e & 3]);
        }
        if (edge) {
          const int lo = window > 0 ? max(0, at - window + 1) : 0;
          const int hi = causal ? min(keys.len, at + 1) : keys.len;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = base + 16 * (e >> 2) + (e & 3);
            if (key < lo || key >= hi) s[rt][e >> 2][e & 3] = -INFINITY;
          }
        }
        if (hide) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = min(max(base + 16 * (e >> 2) + (e & 3), keys.lo), keys.len - 1);
            if ((hide >> ((key >> a.page_shift) - hide0)) & 1) s[rt][e >> 2][e & 3] = -INFINITY;
          }
        }
        float mloc = s[rt][0][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mloc = fmaxf(mloc, s[rt][e >> 2][e & 3]);
        mloc = max_quarters(mloc);
        if (__any(mloc > m_raw[rt] + thr_raw)) {
          const float m_new = fmaxf(m_raw[rt], mloc);
          const float corr = m_raw[rt] == -INFINITY ? 0.f : fast_exp2((m_raw[rt] - m_new) * c);
          l[rt] *= corr;
#pragma unroll
          for (int cb = 0; cb < D / 16; ++cb) oacc[rt][cb] *= corr;
          m_raw[rt] = m_new;
        }
        const float m_use = m_raw[rt] == -INFINITY ? 0.f : m_raw[rt];
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = fast_exp2((s[rt][e >> 2][e & 3] - m_use) * c);
          ls[e & 3] += p;
          const half_t p16 = to16<true>(p);
          pb[rt][e >> 3][e & 7] = p16;
          if constexpr (T::kTwoP) rest[rt][e >> 3][e & 7] = to16<true>(p - from16<true>(p16));
        }
        l[rt] += (ls[0] + ls[1]) + (ls[2] + ls[3]);
      }
      // V's block as bf16 to LDS; values of keys that no row sees become zero.
      const bool part = j * 64 < keys.lo || j * 64 + 64 > keys.len || hide;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int u = lane + 64 * i, key = u / kBlocks, blk = u % kBlocks;
        u32x4 codes = vc[i];
        float scale = scale_of(vs[i]);
        if (part) {
          const int x = j * 64 + key, y = min(max(x, keys.lo), keys.len - 1);
          if (x != y || ((hide >> ((y >> a.page_shift) - hide0)) & 1)) {
            codes = u32x4{0u, 0u, 0u, 0u};
            scale = 1.f;
          }
        }
        char* to = my_v + key * T::kStride + 64 * blk;
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<half8*>(to + 16 * e) = values(codes[e], scale);
      }
      load_v(more ? j + 1 : j, more);
      // (row 4 g + t of 16 keys at columns 4 a .. 4 a + 3 of 16, lane = 16 g + 4 t + a)
      const half_t* from_v =
          reinterpret_cast<const half_t*>(my_v + (4 * g + (l16 >> 2)) * T::kStride + 8 * (l16 & 3));
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int cb = 0; cb < D / 16; ++cb) {
          const half4 lo = lds_read_tr(from_v + 32 * u * (T::kStride / 2) + 16 * cb);
          const half4 hi = lds_read_tr(from_v + (32 * u + 16) * (T::kStride / 2) + 16 * cb);
          const half8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            oacc[rt][cb] = mfma_bf16(v, pb[rt][u], oacc[rt][cb]);
            if constexpr (T::kTwoP) oacc[rt][cb] = mfma_bf16(v, rest[rt][u], oacc[rt][cb]);
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
    // One item: the waves' parts meet in LDS, a row tile at a time, in the accumulator's
    // order: float4 cb * 64 + lane.
    const bool whole = wg1 - wg0 == units;
    if (whole) owned.w = 0;
    if (lane == 0) ra.owned[wg * kLine + wave] = owned;
    slot = 2 * (size_t)(wg * kLine);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      __syncthreads();
      float* const mine = reinterpret_cast<float*>(my_v);
#pragma unroll
      for (int cb = 0; cb < D / 16; ++cb)
        *reinterpret_cast<floatx4*>(mine + (cb * 64 + lane) * 4) = oacc[rt][cb];
      ml[wave * 64 + lane] = make_float2(m_raw[rt], l[rt]);
      __syncthreads();
      float m_star = -INFINITY, l_star = 0.f, wk[kLine];
#pragma unroll
      for (int k = 0; k < kLine; ++k) m_star = fmaxf(m_star, ml[k * 64 + lane].x);
#pragma unroll
      for (int k = 0; k < kLine; ++k) {
        const float m = ml[k * 64 + lane].x;
        wk[k] = m == -INFINITY ? 0.f : fast_exp2((m - m_star) * c);
        l_star += wk[k] * ((ml[k * 64 + l16].y + ml[k * 64 + l16 + 16].y) +
                           (ml[k * 64 + l16 + 32].y + ml[k * 64 + l16 + 48].y));
      }
      const int lr = 16 * rt + l16;
      const Row<T::kRows> row(ra, hkv, tile, lr);
      if (!row.ok) continue;
      const float inv = l_star > 0.f ? 1.f / l_star : 0.f;
      for (int cb = wave; cb < D / 16; cb += kLine) {
        floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kLine; ++k)
          acc += *reinterpret_cast<const floatx4*>(
                     reinterpret_cast<const float*>(vt + k * T::kTileBytes) + (cb * 64 + lane) * 4) * wk[k];
        put(row, whole, lr, inv, 16 * cb + 4 * g, acc);
      }
      if (wave == 0 && g == 0) finish(row, whole, lr, m_star, l_star);
    }
    return;
  } while (pos < end);
  if (lane == 0) late_args().owned[wg * kLine + wave] = owned;
}

// Row tiles that a wave takes: all of a kv head's up to four, of bf16 rows at most 128
// wide, else two (fp16 rows take twice the registers, wide ones too).
template <int D, bool BF>
constexpr int kMostTiles = BF && D <= 128 ? 4 : 2;
template <int D, bool BF, class F>
auto by_row_tiles(int rows, const F& f) {
  if (rows <= 16) return f(Paged4<D, BF, 1>{});
  if constexpr (kMostTiles<D, BF> == 4)
    if (rows > 32) return f(Paged4<D, BF, 4>{});
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
    auto launch = [&](auto full) {
      constexpr bool kFull = decltype(full)::value;
      hipLaunchKernelGGL((paged4_kernel<T, kFull>), dim3(T::kGrid), dim3(T::kThreads), 0,
                         (hipStream_t)a.stream, d);
      const hipError_t e = hipGetLastError();
      return e != hipSuccess ? e : launch_paged_join<T, kFull>(d, (hipStream_t)a.stream);
    };
    if constexpr (T::kD == 256)
      if (a.D != T::kD) return launch(std::false_type{});
    return launch(std::true_type{});
  });
}

}  // namespace fa
