// Torch binding `fa_p100_ext`: the drop-in for the reference's pybind module
// (fa_p100_ext.cu:144-147), with the same two functions, argument lists,
// checks, error messages, allocations and return dtypes:
//
//   forward(q, k, v, causal, full_precision) -> [o fp16 (B,Hq,N,D), lse fp32 (B,Hq,N)]
//       fa_p100_ext.cu:53-83
//   backward(q, k, v, dO, o, lse, causal)    -> [dq fp32 (B,Hq,N,D), dk fp16, dv fp16]
//       fa_p100_ext.cu:103-142
//
// and, with no counterpart in the reference, entries used by the autograd
// Function: backward_half_dq (dq as fp16), forward_bnhd / backward_bnhd
// (dense (B, N, H, D) tensors) and forward_dt / backward_dt (fp16 or bf16);
// the last four take bf16 as well as fp16; pack_mask bit-packs a boolean
// mask for their `mask` / `mask_t` arguments and dropout_bits draws the keep
// bits for `drop` / `drop_t`; they also take an fp32 attention `bias` (and
// the backward its gradient buffer `dbias`). segment_bounds finds packed
// sequences' bounds, and flash_attn is the autograd Function over these entries
// for the calls that need no packed mask, dropout, bias or block lists.
// paged_tables, paged_append and paged_attn are a serving step over a paged
// key/value cache of 16 or 4 bits, paged_gather reads rows of it back, and
// paged_weights and paged_evict cut it to its newest and heaviest keys; all
// without gradients.
//
// Plain C++ (no device code): every launch goes through the C ABI of
// libfa_mi355x.so (include/fa_mi355x.h). Unlike the reference, which uses the
// legacy default stream without a device guard (flash_fwd.cuh:351,
// flash_bwd.cuh:475-483), launches go to torch's current stream on the
// tensors' device.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <vector>

#include "fa_mi355x.h"

namespace {

void check_in(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kHalf, name, " must be fp16");
  TORCH_CHECK(t.dim() == 4, name, " must be (B, H, N, D)");
}

// The entry points added here beside the reference's (forward_dt,
// backward_dt, forward_bnhd, backward_bnhd) also take bf16: q, k, v (and dO,
// o) in one 16-bit format, results in that format.
void check_in16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name,
              " must be fp16 or bf16");
  TORCH_CHECK(t.dim() == 4, name, " must be (B, H, N, D)");
}

// Optional key lengths (right padding): int32 (B,) on q's device; nullptr
// when absent.
const int* kv_len_ptr(const c10::optional<at::Tensor>& kv_len, const at::Tensor& q, int B) {
  if (!kv_len.has_value()) return nullptr;
  const at::Tensor& t = *kv_len;
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), "kv_len must be on q's device");
  TORCH_CHECK(t.scalar_type() == at::kInt, "kv_len must be int32");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == B && t.is_contiguous(), "kv_len must be (B,)");
  return t.data_ptr<int>();
}

int dtype_code(const at::Tensor& q) {
  return q.scalar_type() == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16;
}

// Optional ALiBi slopes: fp32 (Hq,) on q's device; nullptr when absent.
const float* alibi_ptr(const c10::optional<at::Tensor>& slopes, const at::Tensor& q, int H) {
  if (!slopes.has_value()) return nullptr;
  const at::Tensor& t = *slopes;
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), "alibi_slopes must be on q's device");
  TORCH_CHECK(t.scalar_type() == at::kFloat, "alibi_slopes must be fp32");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == H && t.is_contiguous(), "alibi_slopes must be (Hq,)");
  return t.data_ptr<float>();
}

// Optional packed-sequence bounds: int32 (B, N) on q's device; nullptr when absent.
const int* seg_ptr(const c10::optional<at::Tensor>& seg, const at::Tensor& q, int B, int N,
                   const char* name) {
  if (!seg.has_value()) return nullptr;
  const at::Tensor& t = *seg;
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on q's device");
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == B && t.size(1) == N && t.is_contiguous(), name,
              " must be (B, N)");
  return t.data_ptr<int>();
}

// Optional bit-packed mask (pack_mask's output): int32 (B, 1 or Hq, N,
// ceil(N/32)) on q's device; nullptr when absent. Sets *heads to dim 1.
const uint32_t* mask_ptr(const c10::optional<at::Tensor>& m, const at::Tensor& q, int B, int H,
                         int N, const char* name, int* heads) {
  if (!m.has_value()) return nullptr;
  const at::Tensor& t = *m;
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on q's device");
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32 (packed bits)");
  TORCH_CHECK(t.dim() == 4 && t.size(0) == B && (t.size(1) == 1 || t.size(1) == H) &&
                  t.size(2) == N && t.size(3) == (N + 31) / 32 && t.is_contiguous(),
              name, " must be (B, 1 or Hq, N, ceil(N/32))");
  *heads = (int)t.size(1);
  return reinterpret_cast<const uint32_t*>(t.data_ptr<int>());
}

fa_options make_opts(const at::Tensor& q, int layout, const c10::optional<at::Tensor>& kv_len,
                     int64_t window, const c10::optional<at::Tensor>& alibi,
                     const c10::optional<at::Tensor>& seg_start,
                     const c10::optional<at::Tensor>& seg_end, double scale,
                     const c10::optional<at::Tensor>& mask,
                     const c10::optional<at::Tensor>& mask_t,
                     const c10::optional<at::Tensor>& drop,
                     const c10::optional<at::Tensor>& drop_t, double drop_scale,
                     const c10::optional<at::Tensor>& bias,
                     const c10::optional<at::Tensor>& dbias,
                     const c10::optional<at::Tensor>& block_rows,
                     const c10::optional<at::Tensor>& block_cols, int B, int H, int Hkv, int N) {
  fa_options op{};
  op.dtype = dtype_code(q);
  op.layout = layout;
  op.kv_len = kv_len_ptr(kv_len, q, B);
  op.window = (int)window;
  op.alibi_slopes = alibi_ptr(alibi, q, H);
  op.seg_start = seg_ptr(seg_start, q, B, N, "seg_start");
  op.seg_end = seg_ptr(seg_end, q, B, N, "seg_end");
  op.scale = (float)scale;
  int heads = 0, heads_t = 0;
  op.mask = mask_ptr(mask, q, B, H, N, "mask", &heads);
  op.mask_t = mask_ptr(mask_t, q, B, H, N, "mask_t", &heads_t);
  TORCH_CHECK(!op.mask_t || (op.mask && heads_t == heads), "mask_t must come with a mask of its shape");
  op.mask_heads = heads;
  int dheads = 0, dheads_t = 0;
  op.drop = mask_ptr(drop, q, B, H, N, "drop", &dheads);
  op.drop_t = mask_ptr(drop_t, q, B, H, N, "drop_t", &dheads_t);
  TORCH_CHECK(!op.drop || dheads == H, "drop must hold one plane per query head");
  TORCH_CHECK(!op.drop_t || (op.drop && dheads_t == H), "drop_t must come with drop");
  op.drop_scale = (float)drop_scale;
  if (bias.has_value()) {
    // fp32 (B or 1, Hq or 1, N, N) with dense rows; a dimension of size 1 is
    // shared (stride 0).
    const at::Tensor& t = *bias;
    TORCH_CHECK(t.is_cuda() && t.device() == q.device(), "bias must be on q's device");
    TORCH_CHECK(t.scalar_type() == at::kFloat, "bias must be fp32");
    TORCH_CHECK(t.dim() == 4 && (t.size(0) == B || t.size(0) == 1) &&
                    (t.size(1) == H || t.size(1) == 1) && t.size(2) == N && t.size(3) == N &&
                    t.stride(3) == 1 && t.stride(2) == N,
                "bias must be (B or 1, Hq or 1, N, N) with dense rows");
    op.bias = t.data_ptr<float>();
    op.bias_stride_b = t.size(0) == 1 ? 0 : t.stride(0);
    op.bias_stride_h = t.size(1) == 1 ? 0 : t.stride(1);
  }
  if (dbias.has_value()) {
    const at::Tensor& t = *dbias;
    TORCH_CHECK(t.is_cuda() && t.device() == q.device(), "dbias must be on q's device");
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 4 && t.size(0) == B &&
                    t.size(1) == H && t.size(2) == N && t.size(3) == N && t.is_contiguous(),
                "dbias must be fp32 (B, Hq, N, N), contiguous");
    op.dbias = t.data_ptr<float>();
  }
  // Block-sparse lists (pack_blocks): int32 on q's device, of the sizes the
  // shape gives.
  const int64_t nb = (N + FA_SPARSE_BLOCK - 1) / FA_SPARSE_BLOCK;
  auto blocks_ptr = [&](const c10::optional<at::Tensor>& t, int64_t numel, const char* name) {
    if (!t.has_value()) return (const int*)nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == q.device(), name, " must be on q's device");
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous() && t->numel() == numel, name,
                " must be pack_blocks' contiguous int32 list for this shape");
    return (const int*)t->data_ptr<int>();
  };
  op.block_rows = blocks_ptr(block_rows, (int64_t)B * H * nb * (nb + 1), "block_rows");
  op.block_cols =
      blocks_ptr(block_cols, (int64_t)B * Hkv * nb * ((H / Hkv) * nb + 1), "block_cols");
  return op;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FA_OK, what, " failed: ", fa_error_string(rc));
}

void* current_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

}  // namespace

std::vector<at::Tensor> fa_forward(at::Tensor q, at::Tensor k, at::Tensor v, bool causal,
                                   bool full_precision) {
  check_in(q, "q");
  check_in(k, "k");
  check_in(v, "v");
  q = q.contiguous();
  k = k.contiguous();
  v = v.contiguous();
  const int B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int Hkv = k.size(1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads (", H,
              ") must be a multiple of key/value heads (", Hkv, ")");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must match");
  TORCH_CHECK(k.size(0) == B && k.size(2) == N && k.size(3) == D,
              "k/v must be (B, Hkv, N, D) matching q's B, N, D");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(),
              "q, k and v must be on the same device");

  c10::DeviceGuard guard(q.device());
  auto o = at::empty_like(q);
  auto lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  check_rc(fa_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                  B, H, Hkv, N, D, causal ? 1 : 0, full_precision ? 1 : 0, current_stream(q)),
           "fa_fwd");
  return {o, lse};
}

// fa_fwd_ws with a workspace from torch's allocator where the call needs one.
static void forward_ws(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& o, const at::Tensor& lse, int B, int H, int Hkv, int N,
                       int D, bool causal, const fa_options& op) {
  const size_t bytes = fa_fwd_workspace_bytes(B, H, Hkv, N, D, causal ? 1 : 0, &op);
  at::Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check_rc(fa_fwd_ws(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                     bytes ? ws.data_ptr() : nullptr, bytes, B, H, Hkv, N, D, causal ? 1 : 0, &op,
                     current_stream(q)),
           "fa_fwd_ws");
}

// half_dq: dq comes back as fp16 (the fp32 result rounded to nearest even,
// bit-identical to casting the fp32 dq) for the autograd backward, which
// returns dq in q's dtype (fa_p100.py:45); otherwise fp32 as the reference.
static std::vector<at::Tensor> backward_impl(at::Tensor q, at::Tensor k, at::Tensor v,
                                             at::Tensor dO, at::Tensor o, at::Tensor lse,
                                             bool causal, bool half_dq) {
  check_in(q, "q");
  check_in(dO, "dO");
  q = q.contiguous();
  k = k.contiguous();
  v = v.contiguous();
  dO = dO.contiguous();
  o = o.contiguous();
  lse = lse.contiguous();
  const int B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int Hkv = k.size(1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads must be a multiple of kv heads");
  // The reference checks only q and dO here (fa_p100_ext.cu:106); the kernels
  // would read out of bounds on anything else, so the rest is checked too.
  TORCH_CHECK(k.scalar_type() == at::kHalf && v.scalar_type() == at::kHalf &&
                  o.scalar_type() == at::kHalf,
              "k, v and o must be fp16");
  TORCH_CHECK(lse.scalar_type() == at::kFloat, "lse must be fp32");
  TORCH_CHECK(k.sizes() == v.sizes() && k.dim() == 4 && k.size(0) == B && k.size(2) == N &&
                  k.size(3) == D,
              "k/v must be (B, Hkv, N, D) matching q's B, N, D");
  TORCH_CHECK(dO.sizes() == q.sizes() && o.sizes() == q.sizes(), "dO and o must match q");
  TORCH_CHECK(lse.dim() == 3 && lse.size(0) == B && lse.size(1) == H && lse.size(2) == N,
              "lse must be (B, H, N)");

  c10::DeviceGuard guard(q.device());
  auto f32 = q.options().dtype(at::kFloat);
  // Same dtypes as the reference: dq fp32, dk/dv fp16 (fa_p100_ext.cu:118-123).
  auto dq = at::empty({B, H, N, D}, half_dq ? q.options() : f32);
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(k);
  const size_t ws_bytes = fa_bwd_workspace_bytes(B, H, Hkv, N, D);
  auto dvec = at::empty({(int64_t)(ws_bytes / sizeof(float))}, f32);  // rowsum(dO * O)
  if (half_dq)
    check_rc(fa_bwd_half_dq(q.data_ptr(), k.data_ptr(), v.data_ptr(), dO.data_ptr(),
                            o.data_ptr(), lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                            dv.data_ptr(), dvec.data_ptr(), ws_bytes, B, H, Hkv, N, D,
                            causal ? 1 : 0, current_stream(q)),
             "fa_bwd_half_dq");
  else
    check_rc(fa_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), dO.data_ptr(), o.data_ptr(),
                    lse.data_ptr<float>(), dq.data_ptr<float>(), dk.data_ptr(), dv.data_ptr(),
                    dvec.data_ptr(), ws_bytes, B, H, Hkv, N, D, causal ? 1 : 0,
                    current_stream(q)),
             "fa_bwd");
  return {dq, dk, dv};
}

std::vector<at::Tensor> fa_backward(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor dO,
                                    at::Tensor o, at::Tensor lse, bool causal) {
  return backward_impl(q, k, v, dO, o, lse, causal, false);
}

std::vector<at::Tensor> fa_backward_half_dq(at::Tensor q, at::Tensor k, at::Tensor v,
                                            at::Tensor dO, at::Tensor o, at::Tensor lse,
                                            bool causal) {
  return backward_impl(q, k, v, dO, o, lse, causal, true);
}

// The (B, N, H, D)-layout pair used by the autograd Function when q, k, v
// arrive as (B, H, N, D) views of (B, N, H, D) storage (what the HF hook
// passes, fa_p100_hf.py:131-140): no copy in, o and the gradients come back
// in the same layout (dq as fp16). Arguments here are the (B, N, H, D)
// tensors themselves; the checks and messages are the reference's, on the
// logical (B, H, N, D) shapes.
static void check_bnhd(const at::Tensor& t, const char* name) {
  check_in16(t, name);
  TORCH_CHECK(t.is_contiguous(), name, " must be dense (B, N, H, D)");
}

std::vector<at::Tensor> fa_forward_bnhd(at::Tensor q, at::Tensor k, at::Tensor v, bool causal,
                                        c10::optional<at::Tensor> kv_len, int64_t window,
    c10::optional<at::Tensor> alibi_slopes,
    c10::optional<at::Tensor> seg_start, c10::optional<at::Tensor> seg_end,
    double scale, c10::optional<at::Tensor> mask, c10::optional<at::Tensor> mask_t,
    c10::optional<at::Tensor> drop, c10::optional<at::Tensor> drop_t, double drop_scale,
    c10::optional<at::Tensor> bias, c10::optional<at::Tensor> dbias,
    c10::optional<at::Tensor> block_rows, c10::optional<at::Tensor> block_cols) {
  check_bnhd(q, "q");
  check_bnhd(k, "k");
  check_bnhd(v, "v");
  const int B = q.size(0), N = q.size(1), H = q.size(2), D = q.size(3);
  const int Hkv = k.size(2);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads (", H,
              ") must be a multiple of key/value heads (", Hkv, ")");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must match");
  TORCH_CHECK(k.size(0) == B && k.size(1) > 0 && k.size(3) == D,
              "k/v must be (B, Hkv, Nk, D) matching q's B and D");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(),
              "q, k and v must be on the same device");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must have one dtype");
  c10::DeviceGuard guard(q.device());
  auto o = at::empty_like(q);
  auto lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  fa_options op =
      make_opts(q, FA_LAYOUT_BNHD, kv_len, window, alibi_slopes, seg_start, seg_end, scale,
                mask, mask_t, drop, drop_t, drop_scale, bias, dbias, block_rows, block_cols,
                B, H, Hkv, N);
  // key rows that differ from the query rows: bottom-right-aligned causal
  op.kv_rows = k.size(1) != N ? (int)k.size(1) : 0;
  forward_ws(q, k, v, o, lse, B, H, Hkv, N, D, causal, op);
  return {o, lse};
}

std::vector<at::Tensor> fa_backward_bnhd(at::Tensor q, at::Tensor k, at::Tensor v,
                                         at::Tensor dO, at::Tensor o, at::Tensor lse,
                                         bool causal, c10::optional<at::Tensor> kv_len,
                                         int64_t window, c10::optional<at::Tensor> alibi_slopes,
    c10::optional<at::Tensor> seg_start, c10::optional<at::Tensor> seg_end,
    double scale, c10::optional<at::Tensor> mask, c10::optional<at::Tensor> mask_t,
    c10::optional<at::Tensor> drop, c10::optional<at::Tensor> drop_t, double drop_scale,
    c10::optional<at::Tensor> bias, c10::optional<at::Tensor> dbias,
    c10::optional<at::Tensor> block_rows, c10::optional<at::Tensor> block_cols) {
  for (auto& tn : {std::make_pair(&q, "q"), std::make_pair(&k, "k"), std::make_pair(&v, "v"),
                   std::make_pair(&dO, "dO"), std::make_pair(&o, "o")})
    check_bnhd(*tn.first, tn.second);
  lse = lse.contiguous();
  const int B = q.size(0), N = q.size(1), H = q.size(2), D = q.size(3);
  const int Hkv = k.size(2);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads must be a multiple of kv heads");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(1) > 0 && k.size(3) == D,
              "k/v must be (B, Hkv, Nk, D) matching q's B and D");
  TORCH_CHECK(dO.sizes() == q.sizes() && o.sizes() == q.sizes(), "dO and o must match q");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.dim() == 3 && lse.size(0) == B &&
                  lse.size(1) == H && lse.size(2) == N,
              "lse must be (B, H, N)");
  for (const at::Tensor* t : {&k, &v, &dO, &o})
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "q, k, v, dO and o must have one dtype");
  c10::DeviceGuard guard(q.device());
  auto dq = at::empty_like(q);  // q's dtype, (B, N, Hq, D)
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(k);
  const size_t ws_bytes = fa_bwd_workspace_bytes(B, H, Hkv, N, D);
  auto ws = at::empty({(int64_t)(ws_bytes / sizeof(float))}, q.options().dtype(at::kFloat));
  fa_options op =
      make_opts(q, FA_LAYOUT_BNHD, kv_len, window, alibi_slopes, seg_start, seg_end, scale,
                mask, mask_t, drop, drop_t, drop_scale, bias, dbias, block_rows, block_cols,
                B, H, Hkv, N);
  // key rows that differ from the query rows: bottom-right-aligned causal
  op.kv_rows = k.size(1) != N ? (int)k.size(1) : 0;
  check_rc(fa_bwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), dO.data_ptr(), o.data_ptr(),
                     lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                     ws.data_ptr(), ws_bytes, B, H, Hkv, N, D, causal ? 1 : 0, &op,
                     current_stream(q)),
           "fa_bwd_ex");
  return {dq, dk, dv};
}

// Dense (B, H, N, D) tensors in fp16 or bf16 (one format for all), results in
// that format, dq included, and optional key lengths kv_len (int32 (B,), right
// padding: entry b has keys [0, kv_len[b])), sliding window (causal: row i
// sees keys (i - window, i]; 0 = none), ALiBi slopes (fp32 (Hq,): score
// -slope |i - j|), packed-sequence bounds, a softmax scale and a bit-packed
// mask (pack_mask's bits; the backward needs bits_t as mask_t too). For fp16
// without these, the same kernels as forward and backward_half_dq.
std::vector<at::Tensor> fa_forward_dt(at::Tensor q, at::Tensor k, at::Tensor v, bool causal,
                                      c10::optional<at::Tensor> kv_len, int64_t window,
    c10::optional<at::Tensor> alibi_slopes,
    c10::optional<at::Tensor> seg_start, c10::optional<at::Tensor> seg_end,
    double scale, c10::optional<at::Tensor> mask, c10::optional<at::Tensor> mask_t,
    c10::optional<at::Tensor> drop, c10::optional<at::Tensor> drop_t, double drop_scale,
    c10::optional<at::Tensor> bias, c10::optional<at::Tensor> dbias,
    c10::optional<at::Tensor> block_rows, c10::optional<at::Tensor> block_cols) {
  check_in16(q, "q");
  check_in16(k, "k");
  check_in16(v, "v");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must have one dtype");
  q = q.contiguous();
  k = k.contiguous();
  v = v.contiguous();
  const int B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int Hkv = k.size(1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads (", H,
              ") must be a multiple of key/value heads (", Hkv, ")");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must match");
  TORCH_CHECK(k.size(0) == B && k.size(2) > 0 && k.size(3) == D,
              "k/v must be (B, Hkv, Nk, D) matching q's B and D");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(),
              "q, k and v must be on the same device");
  c10::DeviceGuard guard(q.device());
  auto o = at::empty_like(q);
  auto lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  fa_options op =
      make_opts(q, FA_LAYOUT_BHND, kv_len, window, alibi_slopes, seg_start, seg_end, scale,
                mask, mask_t, drop, drop_t, drop_scale, bias, dbias, block_rows, block_cols,
                B, H, Hkv, N);
  // key rows that differ from the query rows: bottom-right-aligned causal
  op.kv_rows = k.size(2) != N ? (int)k.size(2) : 0;
  forward_ws(q, k, v, o, lse, B, H, Hkv, N, D, causal, op);
  return {o, lse};
}

std::vector<at::Tensor> fa_backward_dt(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor dO,
                                       at::Tensor o, at::Tensor lse, bool causal,
                                       c10::optional<at::Tensor> kv_len, int64_t window,
    c10::optional<at::Tensor> alibi_slopes,
    c10::optional<at::Tensor> seg_start, c10::optional<at::Tensor> seg_end,
    double scale, c10::optional<at::Tensor> mask, c10::optional<at::Tensor> mask_t,
    c10::optional<at::Tensor> drop, c10::optional<at::Tensor> drop_t, double drop_scale,
    c10::optional<at::Tensor> bias, c10::optional<at::Tensor> dbias,
    c10::optional<at::Tensor> block_rows, c10::optional<at::Tensor> block_cols) {
  check_in16(q, "q");
  check_in16(dO, "dO");
  q = q.contiguous();
  k = k.contiguous();
  v = v.contiguous();
  dO = dO.contiguous();
  o = o.contiguous();
  lse = lse.contiguous();
  const int B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int Hkv = k.size(1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(N > 0, "N must be positive");
  TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "query heads must be a multiple of kv heads");
  for (const at::Tensor* t : {&k, &v, &dO, &o})
    TORCH_CHECK(t->scalar_type() == q.scalar_type(), "q, k, v, dO and o must have one dtype");
  TORCH_CHECK(lse.scalar_type() == at::kFloat, "lse must be fp32");
  TORCH_CHECK(k.sizes() == v.sizes() && k.dim() == 4 && k.size(0) == B && k.size(2) > 0 &&
                  k.size(3) == D,
              "k/v must be (B, Hkv, Nk, D) matching q's B and D");
  TORCH_CHECK(dO.sizes() == q.sizes() && o.sizes() == q.sizes(), "dO and o must match q");
  TORCH_CHECK(lse.dim() == 3 && lse.size(0) == B && lse.size(1) == H && lse.size(2) == N,
              "lse must be (B, H, N)");
  c10::DeviceGuard guard(q.device());
  auto dq = at::empty_like(q);
  auto dk = at::empty_like(k);
  auto dv = at::empty_like(k);
  const size_t ws_bytes = fa_bwd_workspace_bytes(B, H, Hkv, N, D);
  auto ws = at::empty({(int64_t)(ws_bytes / sizeof(float))}, q.options().dtype(at::kFloat));
  fa_options op =
      make_opts(q, FA_LAYOUT_BHND, kv_len, window, alibi_slopes, seg_start, seg_end, scale,
                mask, mask_t, drop, drop_t, drop_scale, bias, dbias, block_rows, block_cols,
                B, H, Hkv, N);
  // key rows that differ from the query rows: bottom-right-aligned causal
  op.kv_rows = k.size(2) != N ? (int)k.size(2) : 0;
  check_rc(fa_bwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), dO.data_ptr(), o.data_ptr(),
                     lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                     ws.data_ptr(), ws_bytes, B, H, Hkv, N, D, causal ? 1 : 0, &op,
                     current_stream(q)),
           "fa_bwd_ex");
  return {dq, dk, dv};
}

// flash_attn's autograd Function for the calls without a mask, dropout, a bias
// or a block layout: what fa_p100.py's _FlashAttnP100 does, forward and backward
// through the same entries above, without Python between them. The backward of
// a small call waited for the interpreter: the pass (forward and backward) at
// B=1 H=4 N=256 D=64 is 30 us on the GPU.
using OptTensor = c10::optional<at::Tensor>;
class FlashAttn : public torch::autograd::Function<FlashAttn> {
  // The options fa_forward / fa_backward_half_dq do not take.
  static bool has_options(const at::Tensor& q, const at::Tensor& k, const OptTensor& kv_len,
                          int64_t window, const OptTensor& alibi, const OptTensor& seg_start,
                          double scale) {
    return q.scalar_type() == at::kBFloat16 || kv_len.has_value() || window != 0 ||
           alibi.has_value() || seg_start.has_value() || scale != 0.0 || k.size(2) != q.size(2);
  }
  static OptTensor loaded(torch::autograd::AutogradContext* ctx, const char* name) {
    const auto it = ctx->saved_data.find(name);
    return it == ctx->saved_data.end() ? OptTensor() : OptTensor(it->second.toTensor());
  }

 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                            const at::Tensor& k, const at::Tensor& v, bool causal,
                            bool full_precision, const OptTensor& kv_len, int64_t window,
                            const OptTensor& alibi, const OptTensor& seg_start,
                            const OptTensor& seg_end, double scale) {
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["scale"] = scale;
    if (kv_len) ctx->saved_data["kv_len"] = *kv_len;
    if (alibi) ctx->saved_data["alibi"] = *alibi;
    if (seg_start) ctx->saved_data["seg_start"] = *seg_start;
    if (seg_end) ctx->saved_data["seg_end"] = *seg_end;
    const OptTensor none;
    // The (B, N, H, D) path when q is not dense (B, H, N, D) but is dense (B, N,
    // H, D), and k, v are too (with one kv head they are dense in both).
    bool bnhd = !q.is_contiguous();
    at::Tensor qb, kb, vb;
    if (bnhd) {
      qb = q.transpose(1, 2);
      kb = k.transpose(1, 2);
      vb = v.transpose(1, 2);
      bnhd = qb.is_contiguous() && kb.is_contiguous() && vb.is_contiguous();
    }
    ctx->saved_data["bnhd"] = bnhd;
    if (bnhd) {
      auto r = fa_forward_bnhd(qb, kb, vb, causal, kv_len, window, alibi, seg_start, seg_end, scale,
                               none, none, none, none, 1.0, none, none, none, none);
      ctx->save_for_backward({qb, kb, vb, r[0], r[1]});
      return r[0].transpose(1, 2);
    }
    auto r = has_options(q, k, kv_len, window, alibi, seg_start, scale)
                 ? fa_forward_dt(q, k, v, causal, kv_len, window, alibi, seg_start, seg_end, scale,
                                 none, none, none, none, 1.0, none, none, none, none)
                 : fa_forward(q, k, v, causal, full_precision);
    ctx->save_for_backward({q, k, v, r[0], r[1]});
    return r[0];
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const bool causal = ctx->saved_data["causal"].toBool();
    const int64_t window = ctx->saved_data["window"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const OptTensor kv_len = loaded(ctx, "kv_len"), alibi = loaded(ctx, "alibi"),
                    seg_start = loaded(ctx, "seg_start"), seg_end = loaded(ctx, "seg_end"), none;
    std::vector<at::Tensor> d;
    if (ctx->saved_data["bnhd"].toBool()) {
      d = fa_backward_bnhd(saved[0], saved[1], saved[2], grads[0].transpose(1, 2).contiguous(),
                           saved[3], saved[4], causal, kv_len, window, alibi, seg_start, seg_end,
                           scale, none, none, none, none, 1.0, none, none, none, none);
      for (auto& t : d) t = t.transpose(1, 2);
    } else if (has_options(saved[0], saved[1], kv_len, window, alibi, seg_start, scale)) {
      d = fa_backward_dt(saved[0], saved[1], saved[2], grads[0].contiguous(), saved[3], saved[4],
                         causal, kv_len, window, alibi, seg_start, seg_end, scale, none, none, none,
                         none, 1.0, none, none, none, none);
    } else {
      d = fa_backward_half_dq(saved[0], saved[1], saved[2], grads[0].contiguous(), saved[3],
                              saved[4], causal);
    }
    const at::Tensor no;
    return {d[0], d[1], d[2], no, no, no, no, no, no, no, no};
  }
};

at::Tensor fa_flash_attn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                         bool full_precision, const OptTensor& kv_len, int64_t window,
                         const OptTensor& alibi_slopes, const OptTensor& seg_start,
                         const OptTensor& seg_end, double scale) {
  return FlashAttn::apply(q, k, v, causal, full_precision, kv_len, window, alibi_slopes, seg_start,
                          seg_end, scale);
}

// Block layout (Bl, Hl, nb, nb) (bool or uint8; Bl in {1, B}, Hl in {1, Hq};
// nonzero = visible) to the lists the kernels step over (see fa_pack_blocks):
// [block_rows (B, Hq, nb, nb + 1) int32, block_cols (B, Hkv, nb, G*nb + 1)].
std::vector<at::Tensor> fa_pack_blocks_t(at::Tensor layout, int64_t B, int64_t Hq, int64_t Hkv,
                                         int64_t N, bool causal) {
  TORCH_CHECK(layout.is_cuda(), "block layout must be a CUDA tensor");
  TORCH_CHECK(layout.scalar_type() == at::kBool || layout.scalar_type() == at::kByte,
              "block layout must be bool or uint8");
  TORCH_CHECK(B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && N > 0 && N <= INT32_MAX,
              "B, Hq, Hkv and N must be positive, Hq a multiple of Hkv");
  const int64_t nb = (N + FA_SPARSE_BLOCK - 1) / FA_SPARSE_BLOCK;
  TORCH_CHECK(layout.dim() == 4 && (layout.size(0) == 1 || layout.size(0) == B) &&
                  (layout.size(1) == 1 || layout.size(1) == Hq) && layout.size(2) == nb &&
                  layout.size(3) == nb,
              "block layout must be (B or 1, Hq or 1, nb, nb) with nb = ceil(N / ",
              FA_SPARSE_BLOCK, ") = ", nb);
  layout = layout.contiguous();
  c10::DeviceGuard guard(layout.device());
  auto opts = layout.options().dtype(at::kInt);
  auto rows = at::empty({B, Hq, nb, nb + 1}, opts);
  auto cols = at::empty({B, Hkv, nb, (Hq / Hkv) * nb + 1}, opts);
  check_rc(fa_pack_blocks(reinterpret_cast<const uint8_t*>(layout.data_ptr()),
                          (int)layout.size(0), (int)layout.size(1), (int)B, (int)Hq, (int)Hkv,
                          (int)N, causal ? 1 : 0, rows.data_ptr<int>(), cols.data_ptr<int>(),
                          current_stream(layout)),
           "fa_pack_blocks");
  return {rows, cols};
}

// (seg_start, seg_end) of packed sequences (fa_segment_bounds).
std::vector<at::Tensor> fa_segment_bounds_t(at::Tensor ids) {
  TORCH_CHECK(ids.is_cuda() && ids.dim() == 2, "segment ids must be a CUDA tensor (B, N)");
  const bool wide = ids.scalar_type() == at::kLong;
  TORCH_CHECK(wide || ids.scalar_type() == at::kInt, "segment ids must be int32 or int64");
  c10::DeviceGuard guard(ids.device());
  auto opts = ids.options().dtype(at::kInt);
  auto start = at::empty({ids.size(0), ids.size(1)}, opts);
  auto end = at::empty({ids.size(0), ids.size(1)}, opts);
  check_rc(fa_segment_bounds(ids.data_ptr(), wide ? 1 : 0, (int)ids.size(0), (int)ids.size(1),
                             ids.stride(0), ids.stride(1), start.data_ptr<int>(),
                             end.data_ptr<int>(), current_stream(ids)),
           "fa_segment_bounds");
  return {start, end};
}

// Dense boolean mask (..., N, N) (nonzero = may attend) to the packed words
// the kernels read: bits (..., N, ceil(N/32)) and, with `transposed`, bits_t
// of the same shape holding the transpose (see fa_pack_mask).
std::vector<at::Tensor> fa_pack_mask_t(at::Tensor dense, bool transposed) {
  TORCH_CHECK(dense.is_cuda(), "mask must be a CUDA tensor");
  TORCH_CHECK(dense.scalar_type() == at::kBool || dense.scalar_type() == at::kByte,
              "mask must be bool or uint8");
  TORCH_CHECK(dense.dim() >= 2 && dense.size(-1) == dense.size(-2) && dense.size(-1) > 0,
              "mask must be (..., N, N)");
  dense = dense.contiguous();
  const int64_t N = dense.size(-1);
  TORCH_CHECK(N <= INT32_MAX, "mask too large");
  const int64_t P = dense.numel() / (N * N);
  TORCH_CHECK(P > 0 && P <= INT32_MAX, "mask must hold at least one plane");
  std::vector<int64_t> shape(dense.sizes().begin(), dense.sizes().end());
  shape.back() = (N + 31) / 32;
  c10::DeviceGuard guard(dense.device());
  auto opts = dense.options().dtype(at::kInt);
  auto bits = at::empty(shape, opts);
  at::Tensor bits_t = transposed ? at::empty(shape, opts) : at::Tensor();
  check_rc(fa_pack_mask(reinterpret_cast<const uint8_t*>(dense.data_ptr()), (int)P, (int)N,
                        reinterpret_cast<uint32_t*>(bits.data_ptr<int>()),
                        transposed ? reinterpret_cast<uint32_t*>(bits_t.data_ptr<int>()) : nullptr,
                        current_stream(dense)),
           "fa_pack_mask");
  if (!transposed) return {bits};
  return {bits, bits_t};
}

// Dropout keep bits for `drop` / `drop_t`: int32 (B, H, N, ceil(N/32)) each on
// the given device, drawn from `seed` with drop probability p (see
// fa_dropout_bits). Without `transposed` only `drop` is drawn (the forward
// reads no other) and the second tensor is undefined (None in Python).
// causal: the bits of keys past each row's diagonal are cleared and not drawn
// (fa_dropout_bits_causal), for causal attention over N keys.
std::vector<at::Tensor> fa_dropout_bits_t(int64_t seed, double p, int64_t B, int64_t H, int64_t N,
                                          int64_t device, bool transposed, bool causal) {
  TORCH_CHECK(p >= 0.0 && p < 1.0, "dropout p must lie in [0, 1), got ", p);
  TORCH_CHECK(B > 0 && H > 0 && N > 0 && B * H <= INT32_MAX && N <= INT32_MAX,
              "dropout bits need positive B, H, N");
  const at::Device dev(at::kCUDA, (c10::DeviceIndex)device);
  c10::DeviceGuard guard(dev);
  auto opts = at::TensorOptions().dtype(at::kInt).device(dev);
  const int64_t W = (N + 31) / 32;
  auto bits = at::empty({B, H, N, W}, opts);
  at::Tensor bits_t;
  if (transposed) bits_t = at::empty({B, H, N, W}, opts);
  check_rc((causal ? fa_dropout_bits_causal : fa_dropout_bits)(
               (uint64_t)seed, (float)p, (int)(B * H), (int)N,
               reinterpret_cast<uint32_t*>(bits.data_ptr<int>()),
               transposed ? reinterpret_cast<uint32_t*>(bits_t.data_ptr<int>()) : nullptr,
               current_stream(bits)),
           causal ? "fa_dropout_bits_causal" : "fa_dropout_bits");
  return {bits, bits_t};
}

// ---------------------------------------------------------------------------
// Paged key/value caches (fa_paged_tables, fa_paged_append, fa_paged_attn).

// An int32 tensor on `dev`, contiguous along its last dimension.
static void check_ints(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.dim() >= 1 && (t.size(-1) <= 1 || t.stride(-1) == 1), name,
              " must be contiguous along its last dimension");
}

static void check_no_grad(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires grad, and paged caches have no backward: call under torch.no_grad()");
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name,
              " has a forward-mode tangent, and paged caches have no derivative");
}

// A tensor has been written behind autograd's back: what was saved of it is stale.
static void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The stride of a dimension that is walked (one of size 1 has any stride).
static int64_t walk(const at::Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

// Whether 16-byte loads can take t's rows: dense, each on a 16-byte boundary.
static bool rows_aligned(const at::Tensor& t) {
  bool ok = (t.size(-1) <= 1 || t.stride(-1) == 1) && ((uintptr_t)t.data_ptr() & 15) == 0;
  for (int64_t i = 0; i < t.dim() - 1; ++i) ok = ok && walk(t, i) * t.element_size() % 16 == 0;
  return ok;
}

static bool is_16bit(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}

typedef c10::optional<at::Tensor> MaybeTensor;

// The cache of k_cache and v_cache, (pages, Hkv, page_size, D) in any order of
// the first three dimensions, laid out alike; the tables are left unset. four: of 4 bits,
// (pages, Hkv, page_size, D / 2) bytes.
static fa_paged_cache paged_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& like,
                                  bool four = false) {
  TORCH_CHECK(k.is_cuda() && k.device() == like.device() && v.device() == like.device(),
              "k_cache and v_cache must be on ", like.device());
  if (four) {
    TORCH_CHECK(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte,
                "with scales k_cache and v_cache must be uint8, two values of 4 bits each");
  } else {
    TORCH_CHECK(k.scalar_type() == like.scalar_type() && v.scalar_type() == like.scalar_type(),
                "k_cache and v_cache must be ", like.scalar_type(), " as the tokens are");
  }
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(),
              "k_cache and v_cache must both be (pages, Hkv, page_size, D)",
              four ? ", D / 2 bytes a row" : "");
  const int64_t page_size = k.size(2);
  TORCH_CHECK(page_size > 0 && (page_size & (page_size - 1)) == 0 && k.size(0) > 0 &&
                  k.size(0) <= INT32_MAX / page_size,
              "k_cache must hold 1 to 2^31 - 1 rows in pages of a power of two, got ", k.sizes());
  bool alike = rows_aligned(k) && rows_aligned(v);
  for (int64_t i = 0; i < 3; ++i) alike = alike && walk(k, i) == walk(v, i);
  TORCH_CHECK(alike,
              "k_cache and v_cache must be laid out alike, with dense rows and every row 16-byte "
              "aligned");
  fa_paged_cache c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.stride_page = walk(k, 0);
  c.stride_head = walk(k, 1);
  c.stride_row = walk(k, 2);
  c.pages = (int)k.size(0);
  c.page_size = (int)page_size;
  return c;
}

// Whether a cache is of 4 bits: k_scale and v_scale come together.
static bool is_four(const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  TORCH_CHECK(k_scale.has_value() == v_scale.has_value(),
              "k_scale and v_scale must be given together");
  return k_scale.has_value();
}

// The scales of a cache in 4 bits, (pages, Hkv, page_size, D / 32) bytes in any order of the
// first three dimensions, laid out alike.
static fa_paged_scales paged_scales(const at::Tensor& k_scale, const at::Tensor& v_scale,
                                    const at::Tensor& k_cache) {
  fa_paged_scales s{};
  for (const auto& tn : {std::make_pair(&k_scale, "k_scale"), std::make_pair(&v_scale, "v_scale")}) {
    const at::Tensor& t = *tn.first;
    TORCH_CHECK(t.device() == k_cache.device() && t.scalar_type() == at::kByte, tn.second,
                " must be uint8 on ", k_cache.device());
    TORCH_CHECK(t.dim() == 4 && t.size(0) == k_cache.size(0) && t.size(1) == k_cache.size(1) &&
                    t.size(2) == k_cache.size(2) && k_cache.size(3) % 16 == 0 &&
                    t.size(3) == k_cache.size(3) / 16,
                tn.second, " must be (pages, Hkv, page_size, D / 32), a byte for 32 values of "
                "k_cache and v_cache (D a multiple of 32), got ", t.sizes());
    TORCH_CHECK(t.size(3) <= 1 || t.stride(3) == 1, tn.second, "'s rows must be dense");
  }
  for (int64_t i = 0; i < 3; ++i)
    TORCH_CHECK(walk(k_scale, i) == walk(v_scale, i), "k_scale and v_scale must be laid out alike");
  s.k = k_scale.data_ptr<uint8_t>();
  s.v = v_scale.data_ptr<uint8_t>();
  s.stride_page = walk(k_scale, 0);
  s.stride_head = walk(k_scale, 1);
  s.stride_row = walk(k_scale, 2);
  return s;
}

// The head dim that a cache's rows hold.
static int64_t cache_dim(const at::Tensor& cache, bool four) { return cache.size(3) * (four ? 2 : 1); }

// [slots (B, max_new) or (tokens,), kv_len (B,), ring (2,)]; block_table and
// free_pages in place (fa_paged_tables).
std::vector<at::Tensor> fa_paged_tables_t(const at::Tensor& block_table, const at::Tensor& old_len,
                                          const at::Tensor& new_len, const at::Tensor& free_pages,
                                          const at::Tensor& ring, int64_t page_size,
                                          const c10::optional<int64_t>& max_new,
                                          const c10::optional<int64_t>& tokens) {
  TORCH_CHECK(block_table.is_cuda(), "block_table must be a CUDA tensor");
  const at::Device dev = block_table.device();
  check_ints(block_table, dev, "block_table");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) > 0 && block_table.size(1) > 0,
              "block_table must be (B, pages per request)");
  const int64_t B = block_table.size(0), M = block_table.size(1);
  TORCH_CHECK(B == 1 || block_table.stride(0) >= M, "block_table's rows must not overlap");
  check_ints(old_len, dev, "old_len");
  check_ints(new_len, dev, "new_len");
  check_ints(free_pages, dev, "free_pages");
  check_ints(ring, dev, "ring");
  TORCH_CHECK(old_len.dim() == 1 && old_len.size(0) == B && new_len.sizes() == old_len.sizes(),
              "old_len and new_len must be (", B, ",)");
  TORCH_CHECK(free_pages.dim() == 1 && free_pages.size(0) > 0 && free_pages.size(0) <= INT32_MAX / 2,
              "free_pages must be a ring of one page index or more");
  TORCH_CHECK(ring.dim() == 1 && ring.size(0) == 2, "ring must be (2,): head and count");
  TORCH_CHECK(page_size > 0 && (page_size & (page_size - 1)) == 0 && M <= (1 << 30) / page_size,
              "page_size must be a power of two, and a request's pages hold at most 2^30 tokens");
  TORCH_CHECK(max_new.has_value() != tokens.has_value(),
              "one of max_new (slots per request) and tokens (packed slots) must be given");
  const int64_t want = tokens ? *tokens : *max_new;
  TORCH_CHECK(want >= 0 && B <= (1 << 20) && want <= INT32_MAX / (tokens ? 1 : B),
              "max_new and tokens must not be negative, and the slots at most 2^31 - 1");
  c10::DeviceGuard guard(dev);
  at::AutoDispatchBelowADInplaceOrView below;  // (no gradient: the allocations skip its layers)
  const auto opts = old_len.options();
  at::Tensor slots = tokens ? at::empty({want}, opts) : at::empty({B, want}, opts);
  at::Tensor kv_len = at::empty({B}, opts), ring_out = at::empty({2}, opts);
  check_rc(fa_paged_tables(block_table.data_ptr<int>(), B == 1 ? M : block_table.stride(0), (int)M,
                           old_len.data_ptr<int>(), new_len.data_ptr<int>(),
                           free_pages.data_ptr<int>(), (int)free_pages.size(0), ring.data_ptr<int>(),
                           (int)page_size, (int)B, tokens ? 0 : (int)want, tokens ? (int)want : -1,
                           slots.data_ptr<int>(), kv_len.data_ptr<int>(), ring_out.data_ptr<int>(),
                           current_stream(block_table)),
           "fa_paged_tables");
  written(block_table);
  written(free_pages);
  return {slots, kv_len, ring_out};
}

// k, v (T, Hkv, D) with slots (T,), or (B, Hkv, N, D) with slots (B, N), into
// the caches (fa_paged_append; with scales fa_paged4_append).
void fa_paged_append_t(at::Tensor k, at::Tensor v, const at::Tensor& k_cache,
                       const at::Tensor& v_cache, at::Tensor slots, const MaybeTensor& k_scale,
                       const MaybeTensor& v_scale) {
  const bool four = is_four(k_scale, v_scale);
  check_no_grad(k, "k");
  check_no_grad(v, "v");
  check_no_grad(k_cache, "k_cache");
  check_no_grad(v_cache, "v_cache");
  for (auto& tn : {std::make_pair(&k, "k"), std::make_pair(&v, "v")}) {
    const at::Tensor& t = *tn.first;
    TORCH_CHECK(t.is_cuda(), tn.second, " must be a CUDA tensor");
    TORCH_CHECK(is_16bit(t), tn.second, " must be fp16 or bf16");
  }
  TORCH_CHECK((k.dim() == 3 || k.dim() == 4) && k.sizes() == v.sizes(),
              "k and v must both be (T, Hkv, D) or (B, Hkv, N, D)");
  const bool flat = k.dim() == 3;  // (T, Hkv, D): T entries of one row
  const int64_t B = k.size(0), Hkv = k.size(1), N = flat ? 1 : k.size(2), D = k.size(-1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(v.device() == k.device(), "k and v must be on the same device");
  const fa_paged_cache cache = paged_cache(k_cache, v_cache, k, four);
  TORCH_CHECK(k_cache.size(1) == Hkv && cache_dim(k_cache, four) == D &&
                  v.scalar_type() == k.scalar_type(),
              "k, v, k_cache and v_cache must have the same heads, head dim and format");
  const fa_paged_scales scales = four ? paged_scales(*k_scale, *v_scale, k_cache) : fa_paged_scales{};
  TORCH_CHECK(slots.device() == k.device() && slots.scalar_type() == at::kInt,
              "slots must be int32 on ", k.device());
  TORCH_CHECK(slots.dim() == (flat ? 1 : 2) && slots.size(0) == B && (flat || slots.size(1) == N),
              "slots must be (T,) for k of (T, Hkv, D) and (B, N) for k of (B, Hkv, N, D)");
  TORCH_CHECK(B <= INT32_MAX && N <= INT32_MAX && B * N <= INT32_MAX && Hkv * D <= INT32_MAX,
              "k and v may hold at most 2^31 - 1 tokens, of 2^31 - 1 elements");
  at::assert_no_internal_overlap(k_cache);  // (expanded ones, whose rows are several tokens')
  at::assert_no_internal_overlap(v_cache);
  if (four) {
    at::assert_no_internal_overlap(*k_scale);
    at::assert_no_internal_overlap(*v_scale);
  }
  if (B * N * Hkv == 0) return;
  c10::DeviceGuard guard(k.device());
  if (!rows_aligned(k)) k = k.clone(at::MemoryFormat::Contiguous);
  if (!rows_aligned(v)) v = v.clone(at::MemoryFormat::Contiguous);
  slots = slots.contiguous();
  const int64_t kn = flat ? 0 : walk(k, 2), vn = flat ? 0 : walk(v, 2);
  if (four) {
    check_rc(fa_paged4_append(k.data_ptr(), v.data_ptr(), walk(k, 0), kn, walk(k, 1), walk(v, 0), vn,
                              walk(v, 1), slots.data_ptr<int>(), &cache, &scales, (int)B, (int)N,
                              (int)Hkv, (int)D, dtype_code(k), current_stream(k)),
             "fa_paged4_append");
    written(*k_scale);
    written(*v_scale);
  } else {
    check_rc(fa_paged_append(k.data_ptr(), v.data_ptr(), walk(k, 0), kn, walk(k, 1), walk(v, 0), vn,
                             walk(v, 1), slots.data_ptr<int>(), &cache, (int)B, (int)N, (int)Hkv,
                             (int)D, current_stream(k)),
             "fa_paged_append");
  }
  written(k_cache);
  written(v_cache);
}

// [k, v]: the rows at `slots` (T,) or (B, N), (T, Hkv, D) or (B, Hkv, N, D) (fa_paged_gather).
std::vector<at::Tensor> fa_paged_gather_t(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                          at::Tensor slots, const MaybeTensor& k_scale,
                                          const MaybeTensor& v_scale, c10::optional<at::ScalarType> dtype) {
  const bool four = is_four(k_scale, v_scale);
  check_no_grad(k_cache, "k_cache");
  check_no_grad(v_cache, "v_cache");
  const fa_paged_cache cache = paged_cache(k_cache, v_cache, k_cache, four);
  TORCH_CHECK(four || is_16bit(k_cache), "k_cache must be fp16 or bf16, or uint8 with scales");
  const fa_paged_scales scales = four ? paged_scales(*k_scale, *v_scale, k_cache) : fa_paged_scales{};
  const at::ScalarType type = dtype.value_or(four ? at::kBFloat16 : k_cache.scalar_type());
  TORCH_CHECK(four ? type == at::kHalf || type == at::kBFloat16 : type == k_cache.scalar_type(),
              "dtype must be ", four ? "fp16 or bf16" : "the cache's", ", got ", type);
  const int64_t Hkv = k_cache.size(1), D = cache_dim(k_cache, four);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(slots.device() == k_cache.device() && slots.scalar_type() == at::kInt,
              "slots must be int32 on ", k_cache.device());
  TORCH_CHECK(slots.dim() == 1 || slots.dim() == 2, "slots must be (T,) or (B, N)");
  const bool flat = slots.dim() == 1;
  const int64_t B = slots.size(0), N = flat ? 1 : slots.size(1);
  TORCH_CHECK(B <= INT32_MAX && N <= INT32_MAX && B * N <= INT32_MAX && Hkv * D <= INT32_MAX,
              "slots may hold at most 2^31 - 1 tokens, of 2^31 - 1 elements");
  c10::DeviceGuard guard(k_cache.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const auto opts = k_cache.options().dtype(type);
  at::Tensor k = flat ? at::empty({B, Hkv, D}, opts) : at::empty({B, Hkv, N, D}, opts);
  at::Tensor v = at::empty_like(k);
  if (k.numel() == 0) return {k, v};
  slots = slots.contiguous();
  check_rc(fa_paged_gather(k.data_ptr(), v.data_ptr(), flat ? Hkv * D : Hkv * N * D, flat ? 0 : D,
                           flat ? D : N * D, slots.data_ptr<int>(), &cache, four ? &scales : nullptr,
                           (int)B, (int)N, (int)Hkv, (int)D, dtype_code(k), current_stream(k)),
           "fa_paged_gather");
  return {k, v};
}

// What the calls of a batch's newest rows over a cache have in common: checks q (B, H, N,
// D), the table and the lengths against the cache's sizes, and fills the tables of `cache`
// and the options. q in a layout that the kernels do not take, or not 16-byte aligned, is copied.
static fa_options paged_rows(at::Tensor& q, fa_paged_cache& cache, int64_t Hkv,
                             const at::Tensor& block_table, const at::Tensor& kv_len, int64_t window,
                             const c10::optional<at::Tensor>& alibi_slopes, double scale) {
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  TORCH_CHECK(B > 0 && N > 0, "B and N must be positive");
  TORCH_CHECK(Hkv > 0 && H > 0 && H % Hkv == 0, "query heads (", H,
              ") must be a multiple of key/value heads (", Hkv, ")");
  check_ints(block_table, q.device(), "block_table");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B && block_table.size(1) > 0 &&
                  (B == 1 || block_table.stride(0) >= block_table.size(1)),
              "block_table must be (", B, ", pages per request)");
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / cache.page_size,
              "a request's pages hold at most 2^30 tokens");
  check_ints(kv_len, q.device(), "kv_len");
  TORCH_CHECK(kv_len.dim() == 1 && kv_len.size(0) == B, "kv_len must be (", B, ",)");
  TORCH_CHECK(B <= INT32_MAX && H * N <= (1 << 24) && H * D <= INT32_MAX, "shape exceeds the kernels' index range");
  fa_options op{};
  op.dtype = dtype_code(q);
  op.window = (int)std::min<int64_t>(window, INT32_MAX);
  op.alibi_slopes = alibi_ptr(alibi_slopes, q, (int)H);
  op.scale = (float)scale;
  if (!q.is_contiguous()) {
    if (q.transpose(1, 2).is_contiguous()) op.layout = FA_LAYOUT_BNHD;
    else q = q.contiguous();
  }
  if ((uintptr_t)q.data_ptr() & 15) q = q.clone();  // (keeps the strides)
  cache.table = block_table.data_ptr<int>();
  cache.table_stride = B == 1 ? block_table.size(1) : block_table.stride(0);
  cache.table_width = (int)block_table.size(1);
  cache.kv_len = kv_len.data_ptr<int>();
  return op;
}

// [o] or [o, lse]: attention of the newest N tokens over the caches (fa_paged_attn, with
// scales fa_paged4_attn). q as forward_dt's, or a (B, H, N, D) view of a dense (B, N,
// H, D) tensor, whose layout o then has too.
std::vector<at::Tensor> fa_paged_attn_t(at::Tensor q, const at::Tensor& k_cache,
                                        const at::Tensor& v_cache, const at::Tensor& block_table,
                                        const at::Tensor& kv_len, bool causal, int64_t window,
                                        c10::optional<at::Tensor> alibi_slopes, double scale,
                                        bool want_lse, const MaybeTensor& k_scale,
                                        const MaybeTensor& v_scale) {
  const bool four = is_four(k_scale, v_scale);
  check_no_grad(q, "q");
  check_no_grad(k_cache, "k_cache");
  check_no_grad(v_cache, "v_cache");
  if (alibi_slopes) {
    check_no_grad(*alibi_slopes, "alibi_slopes");
    alibi_slopes = alibi_slopes->to(at::kFloat).contiguous();
  }
  check_in16(q, "q");
  fa_paged_cache cache = paged_cache(k_cache, v_cache, q, four);
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int64_t Hkv = k_cache.size(1);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(cache_dim(k_cache, four) == D, "k_cache must be (pages, Hkv, page_size, ", D,
              ") as q's head dim is", four ? ", two values a byte" : "");
  const fa_paged_scales scales = four ? paged_scales(*k_scale, *v_scale, k_cache) : fa_paged_scales{};
  c10::DeviceGuard guard(q.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const fa_options op = paged_rows(q, cache, Hkv, block_table, kv_len, window, alibi_slopes, scale);
  at::Tensor o = at::empty_like(q), lse;
  if (want_lse) lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  const size_t bytes =
      four ? fa_paged4_attn_workspace_bytes((int)B, (int)H, (int)Hkv, (int)N, (int)D)
           : fa_paged_attn_workspace_bytes((int)B, (int)H, (int)Hkv, (int)N, (int)D);
  // (from torch's allocator as a tensor's memory is, without the tensor)
  const c10::DataPtr ws = c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes);
  float* const lse_ptr = want_lse ? lse.data_ptr<float>() : nullptr;
  if (four)
    check_rc(fa_paged4_attn(q.data_ptr(), o.data_ptr(), lse_ptr, &cache, &scales, ws.get(), bytes,
                            (int)B, (int)H, (int)Hkv, (int)N, (int)D, causal ? 1 : 0, &op,
                            current_stream(q)),
             "fa_paged4_attn");
  else
    check_rc(fa_paged_attn(q.data_ptr(), o.data_ptr(), lse_ptr, &cache, ws.get(), bytes, (int)B,
                           (int)H, (int)Hkv, (int)N, (int)D, causal ? 1 : 0, &op, current_stream(q)),
             "fa_paged_attn");
  if (want_lse) return {o, lse};
  return {o};
}

// The weights of a cache's keys, (pages, Hkv, page_size) fp32 in any order of storage.
static void check_weights(const at::Tensor& w, const at::Tensor& k_cache) {
  check_no_grad(w, "weights");
  TORCH_CHECK(w.device() == k_cache.device() && w.scalar_type() == at::kFloat,
              "weights must be float32 on ", k_cache.device());
  TORCH_CHECK(w.dim() == 3 && w.size(0) == k_cache.size(0) && w.size(1) == k_cache.size(1) &&
                  w.size(2) == k_cache.size(2),
              "weights must be (pages, Hkv, page_size) as k_cache is, got ", w.sizes());
  at::assert_no_internal_overlap(w);
}

// Adds the newest rows' weights of the keys to `weights` (fa_paged_weights).
void fa_paged_weights_t(at::Tensor q, const at::Tensor& k_cache, const at::Tensor& block_table,
                        const at::Tensor& kv_len, at::Tensor lse, const at::Tensor& weights,
                        bool causal, int64_t window, c10::optional<at::Tensor> alibi_slopes,
                        double scale, bool restart, const MaybeTensor& k_scale) {
  const bool four = k_scale.has_value();
  check_no_grad(q, "q");
  check_no_grad(k_cache, "k_cache");
  check_no_grad(lse, "lse");
  if (alibi_slopes) {
    check_no_grad(*alibi_slopes, "alibi_slopes");
    alibi_slopes = alibi_slopes->to(at::kFloat).contiguous();
  }
  check_in16(q, "q");
  fa_paged_cache cache = paged_cache(k_cache, k_cache, q, four);
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  TORCH_CHECK(cache_dim(k_cache, four) == D, "k_cache must be (pages, Hkv, page_size, ", D,
              ") as q's head dim is", four ? ", two values a byte" : "");
  const fa_paged_scales scales = four ? paged_scales(*k_scale, *k_scale, k_cache) : fa_paged_scales{};
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.dim() == 3 &&
                  lse.size(0) == B && lse.size(1) == H && lse.size(2) == N,
              "lse must be float32 (", B, ", ", H, ", ", N, ") on ", q.device());
  check_weights(weights, k_cache);
  c10::DeviceGuard guard(q.device());
  at::AutoDispatchBelowADInplaceOrView below;
  lse = lse.contiguous();
  const fa_options op = paged_rows(q, cache, k_cache.size(1), block_table, kv_len, window, alibi_slopes, scale);
  check_rc(fa_paged_weights(q.data_ptr(), lse.data_ptr<float>(), &cache, four ? &scales : nullptr,
                            weights.data_ptr<float>(), walk(weights, 0), walk(weights, 1),
                            walk(weights, 2), restart ? 1 : 0, (int)B, (int)H, (int)k_cache.size(1),
                            (int)N, (int)D, causal ? 1 : 0, &op, current_stream(q)),
           "fa_paged_weights");
  written(weights);
}

// Cuts the requests to max_len tokens, in place; their new lengths (fa_paged_evict).
at::Tensor fa_paged_evict_t(const at::Tensor& k_cache, const at::Tensor& v_cache,
                            const at::Tensor& weights, const at::Tensor& block_table,
                            const at::Tensor& kv_len, const at::Tensor& max_len, int64_t recent,
                            const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  const bool four = is_four(k_scale, v_scale);
  check_no_grad(k_cache, "k_cache");
  check_no_grad(v_cache, "v_cache");
  TORCH_CHECK(four || is_16bit(k_cache), "k_cache must be fp16 or bf16, or uint8 with scales");
  fa_paged_cache cache = paged_cache(k_cache, v_cache, k_cache, four);
  const int64_t Hkv = k_cache.size(1), D = cache_dim(k_cache, four);
  TORCH_CHECK(Hkv > 0, "k_cache must have kv heads");
  TORCH_CHECK(D >= 8 && D <= 256 && D % 8 == 0, "head dim must be a multiple of 8 from 8 to 256, got ", D);
  const fa_paged_scales scales = four ? paged_scales(*k_scale, *v_scale, k_cache) : fa_paged_scales{};
  check_weights(weights, k_cache);
  const at::Device dev = k_cache.device();
  check_ints(block_table, dev, "block_table");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) > 0 && block_table.size(1) > 0 &&
                  (block_table.size(0) == 1 || block_table.stride(0) >= block_table.size(1)),
              "block_table must be (B, pages per request)");
  const int64_t B = block_table.size(0);
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / cache.page_size,
              "a request's pages hold at most 2^30 tokens");
  check_ints(kv_len, dev, "kv_len");
  check_ints(max_len, dev, "max_len");
  TORCH_CHECK(kv_len.dim() == 1 && kv_len.size(0) == B && max_len.sizes() == kv_len.sizes(),
              "kv_len and max_len must be (", B, ",)");
  TORCH_CHECK(recent >= 0, "recent must not be negative");
  TORCH_CHECK(B * Hkv <= (1 << 21), "at most 2^21 requests' kv heads");
  at::assert_no_internal_overlap(k_cache);
  at::assert_no_internal_overlap(v_cache);
  if (four) {
    at::assert_no_internal_overlap(*k_scale);
    at::assert_no_internal_overlap(*v_scale);
  }
  c10::DeviceGuard guard(dev);
  at::AutoDispatchBelowADInplaceOrView below;
  cache.table = block_table.data_ptr<int>();
  cache.table_stride = B == 1 ? block_table.size(1) : block_table.stride(0);
  cache.table_width = (int)block_table.size(1);
  cache.kv_len = kv_len.data_ptr<int>();
  at::Tensor new_len = at::empty({B}, kv_len.options());
  const size_t bytes =
      fa_paged_evict_workspace_bytes((int)B, (int)Hkv, cache.table_width, cache.page_size);
  const c10::DataPtr ws = c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes);
  check_rc(fa_paged_evict(&cache, four ? &scales : nullptr, weights.data_ptr<float>(),
                          walk(weights, 0), walk(weights, 1), walk(weights, 2),
                          max_len.data_ptr<int>(), (int)std::min<int64_t>(recent, INT32_MAX),
                          new_len.data_ptr<int>(), ws.get(), bytes, (int)B, (int)Hkv, (int)D,
                          current_stream(k_cache)),
           "fa_paged_evict");
  written(k_cache);
  written(v_cache);
  written(weights);
  if (four) {
    written(*k_scale);
    written(*v_scale);
  }
  return new_len;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("paged_tables", &fa_paged_tables_t, "Block tables and slots from request lengths",
        py::arg("block_table"), py::arg("old_len"), py::arg("new_len"), py::arg("free_pages"),
        py::arg("ring"), py::arg("page_size"), py::arg("max_new"), py::arg("tokens"));
  m.def("paged_append", &fa_paged_append_t, "Writes tokens' keys and values into a paged cache",
        py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none());
  m.def("paged_gather", &fa_paged_gather_t, "Rows of a paged cache by their slots",
        py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("k_scale"),
        py::arg("v_scale"), py::arg("dtype"));
  m.def("paged_attn", &fa_paged_attn_t, "Attention of the newest tokens over a paged cache",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"),
        py::arg("kv_len"), py::arg("causal"), py::arg("window"), py::arg("alibi_slopes"),
        py::arg("scale"), py::arg("want_lse"), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("paged_weights", &fa_paged_weights_t, "Adds the newest rows' attention weights of cached keys",
        py::arg("q"), py::arg("k_cache"), py::arg("block_table"), py::arg("kv_len"), py::arg("lse"),
        py::arg("weights"), py::arg("causal"), py::arg("window"), py::arg("alibi_slopes"),
        py::arg("scale"), py::arg("restart"), py::arg("k_scale"));
  m.def("paged_evict", &fa_paged_evict_t, "Cuts requests to their newest and heaviest keys",
        py::arg("k_cache"), py::arg("v_cache"), py::arg("weights"), py::arg("block_table"),
        py::arg("kv_len"), py::arg("max_len"), py::arg("recent"), py::arg("k_scale"),
        py::arg("v_scale"));
  m.def("dropout_bits", &fa_dropout_bits_t,
        "Dropout keep bits (B, H, N, ceil(N/32)) and their transpose for drop / drop_t",
        py::arg("seed"), py::arg("p"), py::arg("B"), py::arg("H"), py::arg("N"),
        py::arg("device"), py::arg("transposed") = true, py::arg("causal") = false);
  m.def("dropout_scale", [](double p) { return (double)fa_dropout_scale((float)p); },
        "Scale of the kept probabilities for dropout_bits(p): 1 / (1 - the drawn rate)",
        py::arg("p"));
  m.def("pack_blocks", &fa_pack_blocks_t,
        "block-sparse layout (B|1, Hq|1, nb, nb) to the kernels' block lists",
        py::arg("layout"), py::arg("B"), py::arg("Hq"), py::arg("Hkv"), py::arg("N"),
        py::arg("causal"));
  m.def("flash_attn", &fa_flash_attn, "flash_attn's autograd Function", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("causal"), py::arg("full_precision"),
        py::arg("kv_len") = py::none(), py::arg("window") = 0,
        py::arg("alibi_slopes") = py::none(), py::arg("seg_start") = py::none(),
        py::arg("seg_end") = py::none(), py::arg("scale") = 0.0);
  m.def("segment_bounds", &fa_segment_bounds_t,
        "Bounds (seg_start, seg_end) of packed sequences from (B, N) ids", py::arg("ids"));
  m.def("pack_mask", &fa_pack_mask_t,
        "Bit-packs a dense boolean (..., N, N) mask for the mask / mask_t arguments",
        py::arg("mask"), py::arg("transposed") = true);
  m.def("forward", &fa_forward, "FlashAttention forward (gfx950)");
  m.def("backward", &fa_backward, "FlashAttention backward (gfx950)");
  m.def("backward_half_dq", &fa_backward_half_dq,
        "FlashAttention backward (gfx950), dq as fp16 (used by the autograd Function)");
  m.def("forward_bnhd", &fa_forward_bnhd,
        "FlashAttention forward (gfx950) on dense (B, N, H, D) tensors", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("causal"), py::arg("kv_len") = py::none(), py::arg("window") = 0,
        py::arg("alibi_slopes") = py::none(), py::arg("seg_start") = py::none(),
        py::arg("seg_end") = py::none(), py::arg("scale") = 0.0,
        py::arg("mask") = py::none(), py::arg("mask_t") = py::none(),
        py::arg("drop") = py::none(), py::arg("drop_t") = py::none(), py::arg("drop_scale") = 1.0,
        py::arg("bias") = py::none(), py::arg("dbias") = py::none(),
        py::arg("block_rows") = py::none(), py::arg("block_cols") = py::none());
  m.def("backward_bnhd", &fa_backward_bnhd,
        "FlashAttention backward (gfx950) on dense (B, N, H, D) tensors, dq in q's dtype",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("dO"), py::arg("o"), py::arg("lse"),
        py::arg("causal"), py::arg("kv_len") = py::none(), py::arg("window") = 0,
        py::arg("alibi_slopes") = py::none(), py::arg("seg_start") = py::none(),
        py::arg("seg_end") = py::none(), py::arg("scale") = 0.0,
        py::arg("mask") = py::none(), py::arg("mask_t") = py::none(),
        py::arg("drop") = py::none(), py::arg("drop_t") = py::none(), py::arg("drop_scale") = 1.0,
        py::arg("bias") = py::none(), py::arg("dbias") = py::none(),
        py::arg("block_rows") = py::none(), py::arg("block_cols") = py::none());
  m.def("forward_dt", &fa_forward_dt,
        "FlashAttention forward (gfx950) on fp16 or bf16 (B, H, N, D) tensors", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("causal"), py::arg("kv_len") = py::none(), py::arg("window") = 0,
        py::arg("alibi_slopes") = py::none(), py::arg("seg_start") = py::none(),
        py::arg("seg_end") = py::none(), py::arg("scale") = 0.0,
        py::arg("mask") = py::none(), py::arg("mask_t") = py::none(),
        py::arg("drop") = py::none(), py::arg("drop_t") = py::none(), py::arg("drop_scale") = 1.0,
        py::arg("bias") = py::none(), py::arg("dbias") = py::none(),
        py::arg("block_rows") = py::none(), py::arg("block_cols") = py::none());
  m.def("backward_dt", &fa_backward_dt,
        "FlashAttention backward (gfx950) on fp16 or bf16 (B, H, N, D) tensors, dq in q's dtype",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("dO"), py::arg("o"), py::arg("lse"),
        py::arg("causal"), py::arg("kv_len") = py::none(), py::arg("window") = 0,
        py::arg("alibi_slopes") = py::none(), py::arg("seg_start") = py::none(),
        py::arg("seg_end") = py::none(), py::arg("scale") = 0.0,
        py::arg("mask") = py::none(), py::arg("mask_t") = py::none(),
        py::arg("drop") = py::none(), py::arg("drop_t") = py::none(), py::arg("drop_scale") = 1.0,
        py::arg("bias") = py::none(), py::arg("dbias") = py::none(),
        py::arg("block_rows") = py::none(), py::arg("block_cols") = py::none());
}
