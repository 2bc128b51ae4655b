// Attention of the newest tokens of each request over its paged key/value cache
// (tables and cache writes: fa_pages.hip). No counterpart in the reference,
// which has no cache.
//
// Bound: HBM, each K/V row is read once per 32 query rows. As in fa_dec.hip a row
// tile is 32 rows of one kv head (the rows of the query heads of its group, head
// after head), a wave's step is a block of 32 keys of its own LDS tiles, and the
// products are S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16. What is
// different is where the keys are and how they are dealt out:
//   * the lengths are known on the device only, and differ. So all key blocks of
//     the call, request after request, kv head after kv head, tile after tile, lie
//     on one line, which the workgroups divide evenly: each finds its stretch from
//     the sum of the lengths, walks the items (a row tile of a request's kv head)
//     in it, and writes the result of an item that it has whole; the parts of the
//     others meet in paged_merge_kernel. No workgroup waits for a longer one;
//   * a wave's lanes hold the next 64 page indices of its stretch; a block's rows
//     take theirs from there by a lane permutation, so the table is read once in
//     64 pages and the K/V loads (direct to LDS, an address per lane) wait for
//     nothing. Rows outside the request's keys read one of its rows instead: a
//     masked key's P is zero, but zero times what an unused row holds may be NaN.
#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

constexpr int kRows = 32;  // query rows of a tile
constexpr int kKeys = 32;  // keys of a wave's block

template <int D>
struct Paged {
  static constexpr int kWaves = D > 128 ? 4 : 8;
  static constexpr int kThreads = 64 * kWaves;
  using S = Stream<D>;
  static constexpr int kParts = (S::template bytes<kKeys>() + 1023) / 1024;  // loads of a tile
  static constexpr int kTileBytes = kParts * 1024;
  static constexpr int kFloats = kRows * D;  // a partial O
  // Workgroups that share a CU's 160 KB of LDS.
  static constexpr int kPerCu = kWaves * kTileBytes * 2 > 80 * 1024 ? 1 : 2;
  static constexpr int kGrid = kCUs * kPerCu;
  static_assert(kWaves / 2 * kFloats * 4 <= kWaves * kTileBytes, "merge area exceeds the tiles");

  // The row and 16-byte chunk that lane `lane` of load u brings in.
  __device__ __forceinline__ static void place(int u, int lane, int& row, int& chunk) {
    if constexpr (kSwizzled<D>) {
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
  float* part_o;    // (workgroup, 2) x kRows x D: unscaled partial O
  float2* part_ml;  // (workgroup, 2) x kRows: running max (log2 units), row sum
  int B, Hq, group, N, n_tiles, heads_tiles, causal, window, dr;
  float scale_log2;
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

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ int wave_prefix(int x, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Blocks that a workgroup takes of `total`: a round of its waves at least.
template <int D>
__device__ __forceinline__ int share_of(int total) {
  return max(Paged<D>::kWaves, (total + Paged<D>::kGrid - 1) / Paged<D>::kGrid);
}

// Where the line's position `pos` lies: request b, which begins at `start`. The
// lanes sum runs of `per` requests each, then look at the run that holds pos.
// Sets the line's length; false when pos is past it.
template <int D>
__device__ __forceinline__ bool locate(const PagedKernelArgs& a, int lane, int wg, int& pos,
                                       int& end, int& b, int& start) {
  const int per = (a.B + 63) / 64;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int c = lane * per + i;
    if (c < a.B) mine += Keys(a, a.kv_len[c]).blocks * a.heads_tiles;
  }
  const int through = wave_prefix(mine, lane), total = uniform(__shfl(through, 63));
  const int share = share_of<D>(total);
  pos = wg * share;
  if (pos >= total) return false;
  end = min(pos + share, total);
  const int run = 63 - __clzll(__ballot(through - mine <= pos));
  start = uniform(__shfl(through - mine, run));
  for (int c0 = run * per;; c0 += 64) {
    const int c = c0 + lane;
    const int x = c < min(a.B, (run + 1) * per) ? Keys(a, a.kv_len[c]).blocks * a.heads_tiles : 0;
    const int sum = wave_prefix(x, lane), all = uniform(__shfl(sum, 63));
    if (pos < start + all) {
      const int l = __ffsll(__ballot(start + sum > pos)) - 1;
      b = uniform(c0 + l);
      start = uniform(start + __shfl(sum - x, l));
      return true;
    }
    start += all;
  }
}

// A wave's LDS reads so far are done: its tile may be loaded again.
__device__ __forceinline__ void wait_lds() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_sched_barrier(0);
}

// 16 bytes per lane from `from` to LDS at lds + byte_off + 16 * lane.
__device__ __forceinline__ void lds_direct(void* lds, const char* from, uint32_t byte_off) {
  auto* p = (__attribute__((address_space(3))) char*)lds + byte_off;
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)p, 16, 0, 0);
}

template <int D, bool BF>
__global__ __launch_bounds__((Paged<D>::kThreads)) void paged_kernel(const PagedKernelArgs a) {
  using T = Paged<D>;
  using S = typename T::S;
  constexpr int kWaves = T::kWaves, kParts = T::kParts;
  __shared__ __align__(1024) char kt[kWaves * T::kTileBytes];
  __shared__ __align__(1024) char vt[kWaves * T::kTileBytes];
  __shared__ float2 ml[kWaves * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform(tid >> 6);
  __builtin_assume(wave >= 0 && wave < kWaves);
  const int h = lane >> 5, l32 = lane & 31;
  const int wg = xcd_work_index(T::kGrid);
  int pos, end, b, start;
  if (!locate<D>(a, lane, wg, pos, end, b, start)) return;

  const int Hkv = a.Hq / a.group, rows = a.group * a.N;
  typename S::Offsets off;
  off.init(lane, 0);
  char* const my_k = kt + wave * T::kTileBytes;
  char* const my_v = vt + wave * T::kTileBytes;
  int row[kParts], col[kParts];  // (of this lane's loads; columns in bytes)
#pragma unroll
  for (int u = 0; u < kParts; ++u) {
    int chunk;
    T::place(u, lane, row[u], chunk);
    col[u] = chunk < a.dr / 8 ? 16 * chunk : 0;  // (columns past the head dim: never used)
  }
  const float c = a.scale_log2, thr_raw = kRescaleLog2 / c;
  constexpr int kWaitOlder = 0x0F70 | (kParts & 15) | ((kParts >> 4) << 14);

  while (pos < end) {
    const Keys keys(a, a.kv_len[b]);
    const int item = (pos - start) / keys.blocks;
    const int from = pos - start - item * keys.blocks, upto = min(from + end - pos, keys.blocks);
    const int hkv = item / a.n_tiles, tile = item - hkv * a.n_tiles;
    const int r = tile * kRows + l32;  // this lane's row of the kv head
    const bool row_ok = r < rows;
    const int rc = min(r, rows - 1);
    const int hq = hkv * a.group + rc / a.N, n = rc % a.N;
    const half_t* qrow = a.q + b * a.stq.b + hq * a.stq.h + (size_t)n * a.stq.n;
    half8 qb[D / 16];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
      qb[kk] = as_half8(load16(qrow + kk * 16 + h * 8, kk * 16 + h * 8 < a.dr));
    const float alibi_raw = a.alibi ? a.alibi[hq] * kLog2e / c : 0.f;

    // Keys [lo, hi) of this lane's row, and those that every row sees.
    const int at = keys.len - a.N + n, at0 = keys.len - a.N;
    const int lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
    const int hi = a.causal ? min(keys.len, at + 1) : keys.len;
    const int all_lo = a.window > 0 ? max(0, keys.len - a.window) : 0;
    const int all_hi = a.causal ? at0 + 1 : keys.len;

    // This wave's blocks [j, j1), and the page indices around them.
    const int n_blocks = upto - from, per = (n_blocks + kWaves - 1) / kWaves;
    const int j0 = keys.first + from + wave * per;
    const int j1 = keys.len > keys.lo ? min(j0 + per, keys.first + upto) : 0;
    const int* table = a.table + b * a.table_stride;
    const int last_page = max(keys.len - 1, 0) >> a.page_shift;
    int p0 = 0, held = 0;         // pages p0 .. p0 + 63 are in the lanes' `held`
    unsigned long long hidden = 0;  // of those, the ones outside the pool
    const char* base_k = (const char*)(a.k + hkv * a.head_stride);
    const char* base_v = (const char*)(a.v + hkv * a.head_stride);
    long long offs[kParts];  // of the loaded block's rows
    auto key_of = [&](int j, int u) { return min(max(j * kKeys + row[u], keys.lo), keys.len - 1); };
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
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        const int key = key_of(j, u);
        const int page = __shfl(held, (key >> a.page_shift) - p0);
        offs[u] = 2 * (page * a.page_stride + (key & ((1 << a.page_shift) - 1)) * a.row_stride) + col[u];
      }
    };
    auto load = [&](char* array, const char* base) {
#pragma unroll
      for (int u = 0; u < kParts; ++u)
        lds_direct(array, base + offs[u], (uint32_t)(wave * T::kTileBytes + u * 1024));
    };

    floatx16 oacc[D / 32];
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) oacc[cb] = zero16();
    float m_raw = -INFINITY, l = 0.f;
    if (j0 < j1) {
      fetch(j0);
      place(j0);
      load(kt, base_k);
      load(vt, base_v);
    }
    for (int j = j0; j < j1; ++j) {
      const unsigned long long hide = hidden;  // (of block j's pages, from page hide0 on)
      const int hide0 = p0;
      __builtin_amdgcn_s_waitcnt(kWaitOlder);  // K's block is here, V's may be under way
      floatx16 s = zero16();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) s = mfma16<BF>(S::read16(my_k, off, kk), qb[kk], s);
      wait_lds();
      const bool more = j + 1 < j1;
      if (more) {
        place(j + 1);
        load(kt, base_k);
      }
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
      const float neg = m_raw == -INFINITY ? 0.f : -m_raw * c;
      half8 pb[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = fast_exp2(fmaf(s[e], c, neg));
        l += p;
        pb[e >> 3][e & 7] = to16<BF>(p);
      }
      if (more) __builtin_amdgcn_s_waitcnt(kWaitOlder);  // V's block is here, K's next may be under way
      else wait_vmem();
      if (hide) {
#pragma unroll
        for (int u = 0; u < kParts; ++u)
          if ((hide >> ((key_of(j, u) >> a.page_shift) - hide0)) & 1)
            *reinterpret_cast<u32x4*>(my_v + u * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        wait_lds();
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
          oacc[cb] = mfma16<BF>(S::tr_operand(my_v, q, off, cb), pb[q], oacc[cb]);
      wait_lds();
      if (more) load(vt, base_v);
    }

    // The waves' partials meet in LDS.
    __syncthreads();
    auto part_of = [&](int src) {
      return reinterpret_cast<float*>(src < kWaves / 2 ? kt : vt) + src % (kWaves / 2) * T::kFloats;
    };
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const floatx4 v = {oacc[cb][4 * g], oacc[cb][4 * g + 1], oacc[cb][4 * g + 2],
                           oacc[cb][4 * g + 3]};
        *reinterpret_cast<floatx4*>(part_of(wave) + ((cb * 4 + g) * 64 + lane) * 4) = v;
      }
    ml[wave * 64 + lane] = make_float2(m_raw, l);
    __syncthreads();
    float m_star = -INFINITY, l_star = 0.f, wk[kWaves];
#pragma unroll
    for (int k = 0; k < kWaves; ++k) m_star = fmaxf(m_star, ml[k * 64 + lane].x);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float2 x = ml[k * 64 + lane];
      wk[k] = x.x == -INFINITY ? 0.f : fast_exp2((x.x - m_star) * c);
      l_star += wk[k] * (x.y + ml[k * 64 + (lane ^ 32)].y);
    }
    const bool whole = n_blocks == keys.blocks;
    const float inv_l = l_star > 0.f ? 1.f / l_star : 0.f;  // a row without keys: O = 0
    const size_t slot = 2 * (size_t)wg + (from > 0 ? 0 : 1);
    half_t* orow = a.o + b * a.stq.b + hq * a.stq.h + (size_t)n * a.stq.n;
    constexpr int kRuns = D / 8;  // float4 runs per lane, dealt to the waves
#pragma unroll
    for (int i = 0; i < (kRuns + kWaves - 1) / kWaves; ++i) {
      const int run = i * kWaves + wave;
      if (run >= kRuns || !row_ok) break;
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kWaves; ++k)
        acc += *reinterpret_cast<const floatx4*>(part_of(k) + (run * 64 + lane) * 4) * wk[k];
      if (!whole) {
        *reinterpret_cast<floatx4*>(a.part_o + (slot * kRows + l32) * D + 8 * run + 4 * h) = acc;
      } else if (8 * run + 4 * h < a.dr) {
        half4 o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = to16<BF>(acc[e] * inv_l);
        *reinterpret_cast<half4*>(orow + 8 * run + 4 * h) = o4;
      }
    }
    if (wave == 0 && h == 0 && row_ok) {
      if (!whole) a.part_ml[slot * kRows + l32] = make_float2(m_star * c, l_star);
      else if (a.lse)
        a.lse[((size_t)b * a.Hq + hq) * a.N + n] =
            l_star > 0.f ? (m_star * c + __log2f(l_star)) * kLn2 : INFINITY;
    }
    pos += n_blocks;
    if (pos - start == keys.blocks * a.heads_tiles) {
      start = pos;
      ++b;
    }
    __syncthreads();  // (the merge area is the tiles)
  }
}

// Joins the parts of the items that several workgroups share.
template <int D, bool BF>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedKernelArgs a) {
  const int b = blockIdx.x / a.heads_tiles, item = blockIdx.x - b * a.heads_tiles;
  const int lane = threadIdx.x & 63;
  int before = 0, total = 0;
  for (int i = lane; i < a.B; i += 64) {
    const int x = Keys(a, a.kv_len[i]).blocks;
    total += x;
    if (i < b) before += x;
  }
  before = wave_sum(before);
  total = wave_sum(total);
  const int blocks = Keys(a, a.kv_len[b]).blocks, share = share_of<D>(total * a.heads_tiles);
  const int first = before * a.heads_tiles + item * blocks;
  const int w0 = first / share, w1 = (first + blocks - 1) / share;
  if (w0 == w1) return;  // (its workgroup has written it)
  const int hkv = item / a.n_tiles, tile = item - hkv * a.n_tiles;
  const int rows = min(kRows, a.group * a.N - tile * kRows);
  for (int f = threadIdx.x; f < rows * (D / 4); f += 256) {
    const int rr = f / (D / 4), col = 4 * (f - rr * (D / 4));
    const int r = tile * kRows + rr, hq = hkv * a.group + r / a.N, n = r % a.N;
    // Parts: the second slot of the first workgroup, the first slots of the others.
    const float2* ml = a.part_ml + rr;
    float m = ml[(2 * (size_t)w0 + 1) * kRows].x;
#pragma unroll 4
    for (int w = w0 + 1; w <= w1; ++w) m = fmaxf(m, ml[2 * (size_t)w * kRows].x);
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) {
      const size_t slot = 2 * (size_t)w + (w == w0 ? 1 : 0);
      const float2 x = ml[slot * kRows];
      const float f = x.x == -INFINITY ? 0.f : fast_exp2(x.x - m);  // (no key: zeros)
      l += f * x.y;
      acc += *reinterpret_cast<const floatx4*>(a.part_o + (slot * kRows + rr) * D + col) * f;
    }
    const float inv_l = l > 0.f ? 1.f / l : 0.f;
    if (col < a.dr) {
      half4 o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) o4[e] = to16<BF>(acc[e] * inv_l);
      *reinterpret_cast<half4*>(a.o + b * a.stq.b + hq * a.stq.h + (size_t)n * a.stq.n + col) = o4;
    }
    if (col == 0 && a.lse)
      a.lse[((size_t)b * a.Hq + hq) * a.N + n] = l > 0.f ? (m + __log2f(l)) * kLn2 : INFINITY;
  }
}

}  // namespace

template <>
size_t paged_workspace_w<FA_WIDTH, FA_BF>() {
  return (size_t)Paged<FA_WIDTH>::kGrid * 2 * kRows * (FA_WIDTH * sizeof(float) + sizeof(float2));
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
  d.part_o = (float*)a.workspace;
  d.part_ml = (float2*)(d.part_o + (size_t)Paged<D>::kGrid * 2 * kRows * D);
  d.B = a.B;
  d.Hq = a.Hq;
  d.group = a.Hq / a.Hkv;
  d.N = a.N;
  d.n_tiles = (d.group * a.N + kRows - 1) / kRows;
  d.heads_tiles = a.Hkv * d.n_tiles;
  d.causal = a.causal;
  d.window = a.window < d.cap ? a.window : 0;  // (a wider one hides nothing)
  d.dr = a.D;
  d.scale_log2 = kLog2e * (a.scale > 0.f ? a.scale : 1.f / sqrtf((float)a.D));
  d.alibi = a.alibi;
  d.stq = make_strides(a.layout, a.Hq, a.N, a.D);
  hipLaunchKernelGGL((paged_kernel<D, FA_BF>), dim3(Paged<D>::kGrid), dim3(Paged<D>::kThreads), 0,
                     (hipStream_t)a.stream, d);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_merge_kernel<D, FA_BF>), dim3((unsigned)(a.B * d.heads_tiles)), dim3(256),
                     0, (hipStream_t)a.stream, d);
  return hipGetLastError();
}

}  // namespace fa
