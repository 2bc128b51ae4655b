// Attention of the newest tokens of each request over its paged key/value cache
// (tables and cache writes: fa_pages.hip). No counterpart in the reference,
// which has no cache.
//
// A wave per query row: its lanes hold kGroups keys at a time, a group of lanes
// per key with 8 of the head's columns each, and every group keeps a running
// maximum, sum and output of its own keys, combined at the end.
#include "fa_device.h"
#include "fa_launch.h"

namespace fa {
namespace {

constexpr int kWaves = 4;

struct PagedKernelArgs {
  const half_t* q;
  half_t* o;
  float* lse;
  const half_t* k;
  const half_t* v;
  long long page_stride, head_stride, row_stride;
  int pages, page_shift, page_mask;
  const int* table;
  long long table_stride;
  int cap;  // tokens that a table holds
  const int* kv_len;
  int B, Hq, group, N, causal, window, dr;
  float scale_log2;
  const float* alibi;
  Strides stq;
};

template <int D, bool BF>
__global__ __launch_bounds__(64 * kWaves) void paged_kernel(const PagedKernelArgs a) {
  constexpr int kLanes = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32, kGroups = 64 / kLanes;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= (long long)a.B * a.Hq * a.N) return;
  const int n = (int)(row % a.N), h = (int)(row / a.N % a.Hq), b = (int)(row / a.N / a.Hq);
  const int g = lane / kLanes, col = 8 * (lane % kLanes);
  const bool col_ok = col < a.dr;
  const half_t* qrow = a.q + b * a.stq.b + h * a.stq.h + (size_t)n * a.stq.n;
  const half8 qv = as_half8(load16(qrow + col, col_ok));
  const int len = min(max(a.kv_len[b], 0), a.cap), at = len - a.N + n;
  const int hi = a.causal ? min(len, at + 1) : len;
  const int lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
  const float slope = a.alibi ? a.alibi[h] * kLog2e : 0.f;
  const int* table = a.table + b * a.table_stride;
  float m = -INFINITY, l = 0.f, acc[8] = {};
  for (int j0 = lo; j0 < hi; j0 += kGroups) {
    const int j = j0 + g;
    if (j >= hi) continue;
    const int page = table[j >> a.page_shift];
    if (page < 0 || page >= a.pages) continue;
    const long long off = page * a.page_stride + h / a.group * a.head_stride +
                          (j & a.page_mask) * a.row_stride + col;
    const half8 kv = as_half8(load16(a.k + off, col_ok)), vv = as_half8(load16(a.v + off, col_ok));
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(from16<BF>(qv[e]), from16<BF>(kv[e]), s);
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) s += __shfl_xor(s, d, kLanes);
    s = s * a.scale_log2 - slope * fabsf((float)(at - j));
    const float m_new = fmaxf(m, s);
    const float corr = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
    const float p = m_new == -INFINITY ? 0.f : fast_exp2(s - m_new);
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * corr + p * from16<BF>(vv[e]);
    m = m_new;
  }
#pragma unroll
  for (int d = kLanes; d < 64; d <<= 1) {
    const float m_o = __shfl_xor(m, d), l_o = __shfl_xor(l, d), m_new = fmaxf(m, m_o);
    const float w = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
    const float w_o = m_o == -INFINITY ? 0.f : fast_exp2(m_o - m_new);
    l = l * w + l_o * w_o;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * w + __shfl_xor(acc[e], d) * w_o;
    m = m_new;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (g == 0 && col_ok) {
    half8 out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = to16<BF>(acc[e] * inv);
    *reinterpret_cast<half8*>(a.o + b * a.stq.b + h * a.stq.h + (size_t)n * a.stq.n + col) = out;
  }
  if (lane == 0 && a.lse) a.lse[row] = l > 0.f ? (m + __log2f(l)) * kLn2 : INFINITY;
}

}  // namespace

template <>
hipError_t launch_paged_w<FA_WIDTH, FA_BF>(const PagedArgs& a) {
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
  d.page_mask = (1 << a.pool.page_shift) - 1;
  d.table = a.table;
  d.table_stride = a.table_stride;
  d.cap = a.table_width << a.pool.page_shift;
  d.kv_len = a.kv_len;
  d.B = a.B;
  d.Hq = a.Hq;
  d.group = a.Hq / a.Hkv;
  d.N = a.N;
  d.causal = a.causal;
  d.window = a.window < d.cap ? a.window : 0;  // (a wider one hides nothing)
  d.dr = a.D;
  d.scale_log2 = kLog2e * (a.scale > 0.f ? a.scale : 1.f / sqrtf((float)a.D));
  d.alibi = a.alibi;
  d.stq = make_strides(a.layout, a.Hq, a.N, a.D);
  const long long rows = (long long)a.B * a.Hq * a.N;
  hipLaunchKernelGGL((paged_kernel<FA_WIDTH, FA_BF>), dim3((unsigned)((rows + kWaves - 1) / kWaves)),
                     dim3(64 * kWaves), 0, (hipStream_t)a.stream, d);
  return hipGetLastError();
}

}  // namespace fa
