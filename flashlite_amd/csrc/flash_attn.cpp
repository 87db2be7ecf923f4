// PyTorch-ROCm binding of the `flash_attn_wmma` module: the drop-in
// replacement of the reference's csrc/flash_attn.cpp:4-29 (same module name,
// function names, argument names, defaults and return values).
//
// The torch-side half of the reference host entries lives here, with the
// reference's checks in the reference's order and with its messages:
//   forward_flash2: csrc/kernel_flash2.cu:741-767,
//   forward_naive:  csrc/kernel_naive.cu:252-276, 285.
// Then the call goes through the C ABI (include/flashlite_attn.h) on the
// current HIP stream of the tensors' device.  A non-zero status becomes a
// RuntimeError carrying the library's message (the reference's CUDA_CHECK,
// csrc/includes/flash_attn.h:15-22).  Plain C++: compiled by the host
// compiler, no hipify.

#include <torch/extension.h>

// ROCm PyTorch reports HIP devices as device type `cuda`; its HIP guard and
// stream accessors for that case are the "MasqueradingAsCUDA" variants.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <optional>

#include "flashlite_attn.h"

namespace flash_attn {

namespace {

void* current_stream(const torch::Tensor& t) {
  return static_cast<void*>(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

fl_attn_params make_params(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                           torch::Tensor& o, double sm_scale, bool is_causal) {
  fl_attn_params p;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = o.data_ptr();
  p.batch = q.size(0);
  p.heads = q.size(1);
  p.seq_q = q.size(2);
  p.seq_k = k.size(2);
  p.head_dim = q.size(3);
  p.sm_scale = sm_scale;
  p.causal = is_causal ? 1 : 0;
  return p;
}

void check_same_device(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v) {
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(),
              "All tensors must be on the same device");
}

// bf16 and head_dim 128 (`wide`) calls took any `workspace` without looking at
// it while they ran one pass only: one they cannot use is still no error.
bool usable_workspace(const torch::Tensor& ws, const torch::Tensor& q) {
  return ws.is_cuda() && ws.device() == q.device() && ws.is_contiguous() &&
         reinterpret_cast<uintptr_t>(ws.data_ptr()) % 16 == 0;
}

}  // namespace

torch::Tensor flash_attn_forward_naive(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                       double sm_scale, bool is_causal) {
  TORCH_CHECK(q.is_cuda(), "Query tensor must be on CUDA");
  TORCH_CHECK(k.is_cuda(), "Key tensor must be on CUDA");
  TORCH_CHECK(v.is_cuda(), "Value tensor must be on CUDA");

  TORCH_CHECK(q.is_contiguous(), "Query tensor must be contiguous");
  TORCH_CHECK(k.is_contiguous(), "Key tensor must be contiguous");
  TORCH_CHECK(v.is_contiguous(), "Value tensor must be contiguous");

  TORCH_CHECK(q.dtype() == torch::kHalf, "Query tensor must be FP16 (Half)");
  TORCH_CHECK(k.dtype() == torch::kHalf, "Key tensor must be FP16 (Half)");
  TORCH_CHECK(v.dtype() == torch::kHalf, "Value tensor must be FP16 (Half)");

  TORCH_CHECK(q.dim() == 4, "Query tensor must have 4 dimensions [B, H, N, D]");
  TORCH_CHECK(k.dim() == 4, "Key tensor must have 4 dimensions [B, H, N, D]");
  TORCH_CHECK(v.dim() == 4, "Value tensor must have 4 dimensions [B, H, N, D]");

  TORCH_CHECK(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3),
              "Key dimensions must match Query dimensions [B, H, N_k, D]");
  TORCH_CHECK(v.size(0) == q.size(0) && v.size(1) == q.size(1) && v.size(2) == k.size(2) &&
                  v.size(3) == q.size(3),
              "Value dimensions must match Key dimensions [B, H, N_k, D]");
  check_same_device(q, k, v);

  auto out = torch::empty_like(q);

  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  fl_attn_params p = make_params(q, k, v, out, sm_scale, is_causal);
  const int rc = fl_attn_naive_f16(&p, current_stream(q));
  TORCH_CHECK(rc == FL_OK, "FlashLite HIP error: ", fl_attn_last_error());
  return out;
}

torch::Tensor flash_attn_forward_flash2(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                        double sm_scale, bool is_causal,
                                        std::optional<torch::Tensor> out) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous(),
              "All tensors must be contiguous");
  TORCH_CHECK(q.dtype() == torch::kHalf && k.dtype() == torch::kHalf && v.dtype() == torch::kHalf,
              "All tensors must be FP16 (Half)");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "Tensors must be 4D [B, H, N, D]");

  const int64_t batch_size = q.size(0);
  const int64_t num_heads = q.size(1);
  const int64_t head_dim = q.size(3);

  TORCH_CHECK(k.size(0) == batch_size && k.size(1) == num_heads && k.size(3) == head_dim,
              "Key dimensions must match Query dimensions [B, H, N_k, D]");
  TORCH_CHECK(v.size(0) == batch_size && v.size(1) == num_heads && v.size(2) == k.size(2) &&
                  v.size(3) == head_dim,
              "Value dimensions must match Key dimensions [B, H, N_k, D]");
  TORCH_CHECK(head_dim == 64, "FlashLite WMMA kernel currently requires head_dim == 64");
  check_same_device(q, k, v);

  torch::Tensor out_tensor;
  if (out.has_value() && out.value().defined()) {
    out_tensor = out.value();
    TORCH_CHECK(out_tensor.is_cuda() && out_tensor.is_contiguous(),
                "out tensor must be contiguous CUDA tensor");
    TORCH_CHECK(out_tensor.sizes() == q.sizes(), "out tensor shape must match q");
    TORCH_CHECK(out_tensor.dtype() == torch::kHalf, "out tensor dtype must be FP16");
    TORCH_CHECK(out_tensor.device() == q.device(), "out tensor must be on the same device as q");
  } else {
    out_tensor = torch::empty_like(q);
  }

  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  fl_attn_params p = make_params(q, k, v, out_tensor, sm_scale, is_causal);
  const int rc = fl_attn_fwd_f16(&p, current_stream(q));
  TORCH_CHECK(rc == FL_OK, "FlashLite HIP error: ", fl_attn_last_error());
  return out_tensor;
}

// Beyond the reference surface: any [B, H, N, 64] strided views with a
// unit-stride head dimension (e.g. the transpose of a [B, N, H, 64] tensor),
// N_k != N_q (bottom-right causal), optionally the fp32 log-sum-exp
// [B, H, N_q], and split-KV for few query rows over many keys.  Returns
// `out`, or (out, lse) with return_lse.  An omitted `out` is allocated with
// q's layout (empty_like keeps dense strides); an omitted `lse` (with
// return_lse) as a contiguous fp32 [B, H, N_q] tensor.  Passing both keeps
// the call free of allocations (apart from a split-KV workspace, see below).
// num_splits: 0 = the library's choice, 1 = one pass, n > 1 = n key chunks
// (fp16 at head_dim 64).
// A split-KV call needs a workspace: `workspace` (any device tensor of
// enough bytes, reused across calls for an allocation-free loop; calls that
// may overlap on the GPU must not share one) or else one from the caching
// allocator.  bf16 and head_dim 128 (`wide`) take one from the allocator only
// where the call allocates its output or log-sum-exp anyway; with both given
// and no `workspace` they run one pass and allocate nothing, eagerly and under
// capture alike.
py::object flash_attn_forward_flash2_ex(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                        double sm_scale, bool is_causal,
                                        std::optional<torch::Tensor> out, bool return_lse,
                                        int64_t num_splits,
                                        std::optional<torch::Tensor> workspace,
                                        std::optional<torch::Tensor> lse_out) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), "All tensors must be on CUDA");
  const auto dt = q.scalar_type();
  TORCH_CHECK((dt == torch::kHalf || dt == torch::kBFloat16) && k.scalar_type() == dt &&
                  v.scalar_type() == dt,
              "All tensors must be FP16 (Half), or all BF16");
  const bool bf16 = dt == torch::kBFloat16;
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "Tensors must be 4D [B, H, N, D]");
  const int64_t batch_size = q.size(0);
  const int64_t num_heads = q.size(1);
  const int64_t head_dim = q.size(3);
  TORCH_CHECK(k.size(0) == batch_size && k.size(1) == num_heads && k.size(3) == head_dim,
              "Key dimensions must match Query dimensions [B, H, N_k, D]");
  TORCH_CHECK(v.size(0) == batch_size && v.size(1) == num_heads && v.size(2) == k.size(2) &&
                  v.size(3) == head_dim,
              "Value dimensions must match Key dimensions [B, H, N_k, D]");
  TORCH_CHECK(head_dim == 64 || head_dim == 128, "forward_flash2_ex requires head_dim 64 or 128");
  TORCH_CHECK(q.stride(3) == 1 && k.stride(3) == 1 && v.stride(3) == 1,
              "The head dimension must have unit stride");
  check_same_device(q, k, v);

  torch::Tensor out_tensor;
  const bool out_given = out.has_value() && out.value().defined();
  if (out_given) {
    out_tensor = out.value();
    TORCH_CHECK(out_tensor.is_cuda() && out_tensor.stride(3) == 1,
                "out tensor must be a CUDA tensor with a unit-stride head dimension");
    TORCH_CHECK(out_tensor.sizes() == q.sizes(), "out tensor shape must match q");
    TORCH_CHECK(out_tensor.scalar_type() == dt, "out tensor dtype must match q");
    TORCH_CHECK(out_tensor.device() == q.device(), "out tensor must be on the same device as q");
  } else {
    out_tensor = torch::empty_like(q);
  }
  torch::Tensor lse;
  const bool lse_given = lse_out.has_value() && lse_out.value().defined();
  TORCH_CHECK(!lse_given || return_lse, "lse= needs return_lse=True");
  if (lse_given) {
    lse = lse_out.value();
    TORCH_CHECK(lse.is_cuda() && lse.device() == q.device(),
                "lse tensor must be on the same device as q");
    TORCH_CHECK(lse.scalar_type() == torch::kFloat32, "lse tensor dtype must be float32");
    TORCH_CHECK(lse.dim() == 3 && lse.size(0) == batch_size && lse.size(1) == num_heads &&
                    lse.size(2) == q.size(2) && lse.is_contiguous(),
                "lse tensor must be a contiguous [B, H, N_q] tensor");
  } else if (return_lse)
    lse = torch::empty({batch_size, num_heads, q.size(2)},
                       q.options().dtype(torch::kFloat32).memory_format(torch::MemoryFormat::Contiguous));

  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  fl_attn_params_ex p;
  p.base = make_params(q, k, v, out_tensor, sm_scale, is_causal);
  const torch::Tensor* ts[4] = {&q, &k, &v, &out_tensor};
  int64_t* st[4] = {p.q_stride, p.k_stride, p.v_stride, p.o_stride};
  for (int i = 0; i < 4; ++i)
    for (int d = 0; d < 3; ++d) st[i][d] = ts[i]->stride(d);
  p.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  TORCH_CHECK(num_splits >= 0 && num_splits <= INT32_MAX, "num_splits must be >= 0");
  // An explicit chunk count is built for fp16 at head_dim 64; with
  // num_splits 0 the library chooses for every type.
  const bool wide = bf16 || head_dim != 64;
  TORCH_CHECK(!wide || num_splits <= 1,
              "split-KV (num_splits > 1) needs fp16 tensors with head_dim 64");
  const bool allocates = !out_given || (return_lse && !lse_given);
  const int32_t dtype = bf16 ? FL_DTYPE_BF16 : FL_DTYPE_F16;
  const int64_t ws_bytes = num_splits == 1 ? 0
                           : num_splits == 0
                               ? fl_attn_workspace_bytes(&p, dtype)
                               : fl_attn_splitkv_workspace_bytes(&p, (int32_t)num_splits);
  TORCH_CHECK(ws_bytes >= 0, "FlashLite HIP error: ", fl_attn_last_error());
  int rc;
  if (ws_bytes == 0) {
    rc = bf16 ? fl_attn_fwd_bf16_ex(&p, -1, current_stream(q))
              : fl_attn_fwd_f16_ex(&p, -1, current_stream(q));
  } else {
    torch::Tensor ws;
    void* buf = nullptr;
    size_t have = 0;
    if (workspace.has_value() && workspace.value().defined() &&
        workspace.value().nbytes() >= (size_t)ws_bytes &&
        (!wide || usable_workspace(workspace.value(), q))) {
      ws = workspace.value();
      TORCH_CHECK(ws.is_cuda() && ws.device() == q.device() && ws.is_contiguous(),
                  "workspace must be a contiguous tensor on q's device");
      buf = ws.data_ptr();
      have = ws.nbytes();
    } else if (!wide || allocates) {
      ws = torch::empty({(ws_bytes + 3) / 4}, q.options().dtype(torch::kFloat32));
      buf = ws.data_ptr();
      have = ws.nbytes();
    }  // else one pass
    rc = num_splits == 0 ? fl_attn_fwd_ws(&p, dtype, buf, (int64_t)have, current_stream(q))
                         : fl_attn_fwd_f16_splitkv(&p, (int32_t)num_splits, buf, (int64_t)have,
                                                   current_stream(q));
  }
  TORCH_CHECK(rc == FL_OK, "FlashLite HIP error: ", fl_attn_last_error());
  if (return_lse) return py::make_tuple(out_tensor, lse);
  return py::cast(out_tensor);
}


// ---------------------------------------------------------------------------
// Serving over a paged cache (include/flashlite_attn.h has the semantics): no
// counterpart in the reference.

namespace {

using OptTensor = std::optional<torch::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t.value().defined(); }

void check_int32(const torch::Tensor& t, const torch::Device& dev, int64_t dim, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name, " must be on the same device as the others");
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension(s)");
}

// A contiguous [B] int32 tensor.
const int32_t* requests(const torch::Tensor& t, const torch::Device& dev, int64_t batch,
                        const char* name) {
  check_int32(t, dev, 1, name);
  TORCH_CHECK(t.size(0) == batch, name, " must have one entry per request");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  return t.data_ptr<int32_t>();
}

// An output of `shape`: `t` if given, or a new tensor on `dev`.
torch::Tensor output(const OptTensor& t, at::IntArrayRef shape, torch::ScalarType type,
                     const torch::Device& dev, const char* name) {
  if (!given(t)) return torch::empty(shape, torch::TensorOptions().dtype(type).device(dev));
  const torch::Tensor& x = t.value();
  TORCH_CHECK(x.is_cuda() && x.device() == dev, name, " must be on the same device as the others");
  TORCH_CHECK(x.scalar_type() == type && x.sizes() == shape && x.is_contiguous(), name,
              " must be a contiguous ", type, " tensor of shape ", shape);
  return x;
}

int32_t serve_dtype(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kHalf: return FL_DTYPE_F16;
    case torch::kBFloat16: return FL_DTYPE_BF16;
    case torch::kFloat32: return FL_DTYPE_F32;
    default: return -1;
  }
}

// A [B, H, N, D] view: strides {batch, head, row}, unit-stride D.
void view4(const torch::Tensor& t, const torch::Tensor& like, const char* name, int64_t st[3]) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name,
              " must be on the same device as the others");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the dtype of the others");
  TORCH_CHECK(t.dim() == 4, name, " must be 4D");
  TORCH_CHECK(t.stride(3) == 1 || t.size(3) == 1 || t.numel() == 0, name,
              " must have a unit-stride head dimension");
  for (int i = 0; i < 3; ++i) st[i] = t.stride(i);
}

// A [B, N] (or broadcast [N]) tensor's strides.
void view2(const torch::Tensor& t, int64_t batch, int64_t rows, const char* name, int64_t st[2]) {
  if (t.dim() == 1) {
    TORCH_CHECK(t.size(0) == rows, name, " must have one entry per row");
    st[0] = 0;
    st[1] = t.stride(0);
  } else {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == batch && t.size(1) == rows, name,
                " must be [B, N]");
    st[0] = t.stride(0);
    st[1] = t.stride(1);
  }
}

void ok(int rc) { TORCH_CHECK(rc == FL_OK, "FlashLite HIP error: ", fl_attn_last_error()); }

}  // namespace

py::tuple plan_cache(const torch::Tensor& lengths, const torch::Tensor& counts,
                     const torch::Tensor& block_tables, const torch::Tensor& held,
                     const torch::Tensor& free_blocks, const torch::Tensor& free_state,
                     int64_t block_size, int64_t width, const OptTensor& held_out,
                     const OptTensor& state_out, const OptTensor& positions,
                     const OptTensor& slots, const OptTensor& info) {
  TORCH_CHECK(lengths.is_cuda(), "All tensors must be on CUDA");
  const auto dev = lengths.device();
  TORCH_CHECK(lengths.dim() == 1, "lengths must have 1 dimension(s)");
  TORCH_CHECK(block_size >= 1 && width >= 0, "block_size must be positive and width not negative");
  const int64_t batch = lengths.size(0);
  fl_cache_plan_params p;
  p.lengths = requests(lengths, dev, batch, "lengths");
  p.counts = requests(counts, dev, batch, "counts");
  p.held = requests(held, dev, batch, "held");
  p.held_out = const_cast<int32_t*>(
      given(held_out) ? requests(held_out.value(), dev, batch, "held_out") : p.held);
  check_int32(block_tables, dev, 2, "block_tables");
  TORCH_CHECK(block_tables.size(0) == batch && (block_tables.stride(1) == 1 ||
                                                block_tables.size(1) <= 1),
              "block_tables must be [B, M] with unit-stride rows");
  p.block_tables = block_tables.data_ptr<int32_t>();
  check_int32(free_blocks, dev, 1, "free_blocks");
  TORCH_CHECK(free_blocks.is_contiguous() && free_blocks.size(0) >= 1,
              "free_blocks must be contiguous and not empty");
  p.free_blocks = free_blocks.data_ptr<int32_t>();
  p.free_state = requests(free_state, dev, 2, "free_state");
  p.free_state_out = const_cast<int32_t*>(
      given(state_out) ? requests(state_out.value(), dev, 2, "state_out") : p.free_state);
  const torch::Tensor pos = output(positions, {batch, width}, torch::kInt32, dev, "positions");
  const torch::Tensor slot = output(slots, {batch, width}, torch::kInt64, dev, "slots");
  const torch::Tensor inf = output(info, {batch, 4}, torch::kInt32, dev, "info");
  p.positions = pos.data_ptr<int32_t>();
  p.slots = slot.data_ptr<int64_t>();
  p.info = inf.data_ptr<int32_t>();
  p.batch = batch;
  p.width = width;
  p.block_size = block_size;
  p.max_blocks = block_tables.size(1);
  p.table_stride = block_tables.stride(0);
  p.pool = free_blocks.size(0);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  ok(fl_attn_cache_plan(&p, current_stream(lengths)));
  return py::make_tuple(pos, slot, inf);
}

py::tuple plan_tree(const torch::Tensor& parents, const torch::Tensor& lengths,
                    const OptTensor& counts, const OptTensor& mask, const OptTensor& positions) {
  TORCH_CHECK(parents.is_cuda(), "All tensors must be on CUDA");
  const auto dev = parents.device();
  check_int32(parents, dev, 2, "parents");
  TORCH_CHECK(parents.stride(1) == 1 || parents.size(1) <= 1, "parents must have unit-stride rows");
  const int64_t batch = parents.size(0), n = parents.size(1);
  fl_tree_plan_params p;
  p.parents = parents.data_ptr<int32_t>();
  p.lengths = requests(lengths, dev, batch, "lengths");
  p.counts = given(counts) ? requests(counts.value(), dev, batch, "counts") : nullptr;
  const torch::Tensor m = output(mask, {batch, n, (n + 63) / 64}, torch::kInt64, dev, "mask");
  const torch::Tensor pos = output(positions, {batch, n}, torch::kInt32, dev, "positions");
  p.mask = m.data_ptr<int64_t>();
  p.positions = pos.data_ptr<int32_t>();
  p.batch = batch;
  p.drafts = n;
  p.parent_stride = parents.stride(0);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  ok(fl_attn_tree_plan(&p, current_stream(parents)));
  return py::make_tuple(m, pos);
}

namespace {

// q, k (or none), positions and freqs of a rotary call.
fl_rotary_params rotary_params(const torch::Tensor& q, const OptTensor& k,
                               const torch::Tensor& positions, const torch::Tensor& freqs,
                               bool interleaved, double scale) {
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  fl_rotary_params p = {};
  p.dtype = serve_dtype(q);
  TORCH_CHECK(p.dtype >= 0, "All tensors must be FP16 (Half), BF16 or FP32");
  view4(q, q, "q", p.q_stride);
  p.batch = q.size(0);
  p.heads = q.size(1);
  p.rows = q.size(2);
  p.head_dim = q.size(3);
  p.q = q.data_ptr();
  if (given(k)) {
    view4(*k, q, "k", p.k_stride);
    TORCH_CHECK(k->size(0) == p.batch && k->size(2) == p.rows && k->size(3) == p.head_dim,
                "k must be [B, H_k, N, D] with q's B, N and D");
    p.k = k->data_ptr();
    p.kv_heads = k->size(1);
  }
  TORCH_CHECK(positions.is_cuda() && positions.device() == q.device(),
              "positions must be on the same device as the others");
  TORCH_CHECK(positions.scalar_type() == torch::kInt32 || positions.scalar_type() == torch::kInt64,
              "positions must be int32 or int64");
  view2(positions, p.batch, p.rows, "positions", p.position_stride);
  p.positions = positions.data_ptr();
  p.position_bits = positions.scalar_type() == torch::kInt64 ? 64 : 32;
  TORCH_CHECK(freqs.is_cuda() && freqs.device() == q.device() && freqs.dim() == 1 &&
                  freqs.scalar_type() == torch::kFloat64 && freqs.is_contiguous(),
              "freqs must be a contiguous float64 tensor of one dimension on q's device");
  p.freqs = freqs.data_ptr<double>();
  p.pairs = freqs.size(0);
  p.scale = scale;
  p.interleaved = interleaved ? 1 : 0;
  return p;
}

py::object rotary(const torch::Tensor& q, const OptTensor& k, const torch::Tensor& positions,
                  const torch::Tensor& freqs, bool interleaved, double scale,
                  const OptTensor& q_out, const OptTensor& k_out, bool transpose) {
  fl_rotary_params p = rotary_params(q, k, positions, freqs, interleaved, scale);
  p.transpose = transpose ? 1 : 0;
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const torch::Tensor qo = given(q_out) ? *q_out : torch::empty_like(q);
  view4(qo, q, "q_out", p.q_out_stride);
  TORCH_CHECK(qo.sizes() == q.sizes(), "q_out must have q's shape");
  p.q_out = qo.data_ptr();
  torch::Tensor ko;
  if (given(k)) {
    ko = given(k_out) ? *k_out : torch::empty_like(*k);
    view4(ko, q, "k_out", p.k_out_stride);
    TORCH_CHECK(ko.sizes() == k->sizes(), "k_out must have k's shape");
    p.k_out = ko.data_ptr();
  } else {
    TORCH_CHECK(!given(k_out), "k_out= needs k");
  }
  ok(fl_attn_rotary(&p, current_stream(q)));
  if (given(k)) return py::make_tuple(qo, ko);
  return py::cast(qo);
}

}  // namespace

py::object forward_rotary(const torch::Tensor& q, const OptTensor& k,
                          const torch::Tensor& positions, const torch::Tensor& freqs,
                          bool interleaved, double scale, const OptTensor& q_out,
                          const OptTensor& k_out) {
  return rotary(q, k, positions, freqs, interleaved, scale, q_out, k_out, false);
}

py::object backward_rotary(const torch::Tensor& dq, const OptTensor& dk,
                           const torch::Tensor& positions, const torch::Tensor& freqs,
                           bool interleaved, double scale, const OptTensor& q_out,
                           const OptTensor& k_out) {
  return rotary(dq, dk, positions, freqs, interleaved, scale, q_out, k_out, true);
}

namespace {

// The caches and slots of a call that stores k and v.
fl_cache_store cache_store(const fl_rotary_params& p, const torch::Tensor& q,
                           const torch::Tensor& k, const torch::Tensor& v,
                           const torch::Tensor& slots, const torch::Tensor& k_cache,
                           const torch::Tensor& v_cache) {
  TORCH_CHECK(p.dtype != FL_DTYPE_F32, "All tensors must be FP16 (Half), or all BF16");
  fl_cache_store c = {};
  view4(v, q, "v", c.v_stride);
  TORCH_CHECK(v.sizes() == k.sizes(), "v must have k's shape");
  view4(k_cache, q, "k_cache", c.k_cache_stride);
  view4(v_cache, q, "v_cache", c.v_cache_stride);
  TORCH_CHECK(k_cache.size(1) == p.kv_heads && k_cache.size(3) == p.head_dim &&
                  v_cache.sizes() == k_cache.sizes(),
              "The caches must be [blocks, H_k, block_size, D] with k's H_k and D");
  TORCH_CHECK(slots.is_cuda() && slots.device() == q.device() &&
                  slots.scalar_type() == torch::kInt64,
              "slots must be int64 on the same device as the others");
  view2(slots, p.batch, p.rows, "slots", c.slot_stride);
  TORCH_CHECK(slots.dim() == 2 || p.batch == 1, "slots must be [B, N]");
  c.v = v.data_ptr();
  c.k_cache = k_cache.data_ptr();
  c.v_cache = v_cache.data_ptr();
  c.num_blocks = k_cache.size(0);
  c.block_size = k_cache.size(2);
  c.slots = slots.data_ptr<int64_t>();
  return c;
}

// The caller's workspace of at least `need` bytes, or a new one.
torch::Tensor workspace_of(const OptTensor& workspace, int64_t need, const torch::Tensor& like) {
  if (!given(workspace))
    return torch::empty({(need + 3) / 4}, like.options().dtype(torch::kFloat32));
  const torch::Tensor& ws = *workspace;
  TORCH_CHECK(ws.is_cuda() && ws.device() == like.device() && ws.is_contiguous(),
              "workspace must be a contiguous tensor on q's device");
  TORCH_CHECK((int64_t)ws.nbytes() >= need, "workspace of ", need, " bytes needed (got ",
              ws.nbytes(), ")");
  return ws;
}

}  // namespace

torch::Tensor rotary_to_cache(const torch::Tensor& q, const torch::Tensor& k,
                              const torch::Tensor& v, const torch::Tensor& positions,
                              const torch::Tensor& slots, const torch::Tensor& freqs,
                              const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                              bool interleaved, double scale, const OptTensor& out) {
  fl_rotary_params p = rotary_params(q, k, positions, freqs, interleaved, scale);
  const fl_cache_store c = cache_store(p, q, k, v, slots, k_cache, v_cache);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const torch::Tensor o = given(out) ? *out : torch::zeros_like(q);
  view4(o, q, "out", p.q_out_stride);
  TORCH_CHECK(o.sizes() == q.sizes(), "out must have q's shape");
  p.q_out = o.data_ptr();
  ok(fl_attn_rotary_cache(&p, &c, current_stream(q)));
  return o;
}

namespace {

// Weights, epsilon and axes of a call that norms; `positions` with axes is
// [A, B, N] (or [A, N]).
fl_norm_params norm_params(const torch::Tensor& q, const OptTensor& k, const OptTensor& q_weight,
                           const OptTensor& k_weight, const torch::Tensor& positions,
                           const OptTensor& axes, int64_t pairs, double eps, double offset) {
  fl_norm_params n = {};
  n.weight_dtype = FL_DTYPE_F32;
  n.eps = eps;
  n.weight_offset = offset;
  auto weight = [&](const OptTensor& w, const char* name) -> const void* {
    if (!given(w)) return nullptr;
    TORCH_CHECK(w->is_cuda() && w->device() == q.device(), name,
                " must be on the same device as the others");
    TORCH_CHECK(w->scalar_type() == torch::kFloat32 || w->scalar_type() == q.scalar_type(), name,
                " must be FP32 or of q's dtype");
    TORCH_CHECK(w->dim() == 1 && w->size(0) == q.size(3) && w->is_contiguous(), name,
                " must be a contiguous [D] tensor");
    return w->data_ptr();
  };
  n.q_weight = weight(q_weight, "q_weight");
  n.k_weight = weight(k_weight, "k_weight");
  TORCH_CHECK(given(k) || !given(k_weight), "k_weight= needs k");
  if (given(q_weight) && given(k_weight))
    TORCH_CHECK(q_weight->scalar_type() == k_weight->scalar_type(),
                "q_weight and k_weight must have the same dtype");
  if (given(q_weight) || given(k_weight))
    n.weight_dtype = serve_dtype(given(q_weight) ? *q_weight : *k_weight);
  if (given(axes)) {
    check_int32(*axes, q.device(), 1, "axes");
    TORCH_CHECK(axes->size(0) == pairs && axes->is_contiguous(),
                "axes must be contiguous, an axis for each of freqs");
    n.axes = axes->data_ptr<int32_t>();
    n.num_axes = positions.size(0);
    n.axis_stride = positions.stride(0);
  }
  return n;
}

// The positions of the first axis, as rotary_params takes them.
torch::Tensor first_axis(const torch::Tensor& positions, const OptTensor& axes) {
  if (!given(axes)) return positions;
  TORCH_CHECK((positions.dim() == 2 || positions.dim() == 3) && positions.size(0) >= 1,
              "positions must be [A, B, N] or [A, N] with axes");
  return positions.select(0, 0);
}

}  // namespace

py::object forward_norm_rotary(const torch::Tensor& q, const OptTensor& k,
                               const OptTensor& q_weight, const OptTensor& k_weight,
                               const torch::Tensor& positions, const torch::Tensor& freqs,
                               const OptTensor& axes, double eps, double weight_offset,
                               bool interleaved, double scale, const OptTensor& q_out,
                               const OptTensor& k_out) {
  fl_rotary_params p =
      rotary_params(q, k, first_axis(positions, axes), freqs, interleaved, scale);
  const fl_norm_params n =
      norm_params(q, k, q_weight, k_weight, positions, axes, p.pairs, eps, weight_offset);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const torch::Tensor qo = given(q_out) ? *q_out : torch::empty_like(q);
  view4(qo, q, "q_out", p.q_out_stride);
  TORCH_CHECK(qo.sizes() == q.sizes(), "q_out must have q's shape");
  p.q_out = qo.data_ptr();
  torch::Tensor ko;
  if (given(k)) {
    ko = given(k_out) ? *k_out : torch::empty_like(*k);
    view4(ko, q, "k_out", p.k_out_stride);
    TORCH_CHECK(ko.sizes() == k->sizes(), "k_out must have k's shape");
    p.k_out = ko.data_ptr();
  } else {
    TORCH_CHECK(!given(k_out), "k_out= needs k");
  }
  ok(fl_attn_norm_rotary(&p, &n, current_stream(q)));
  if (given(k)) return py::make_tuple(qo, ko);
  return py::cast(qo);
}

py::tuple backward_norm_rotary(const torch::Tensor& dq, const OptTensor& dk, const torch::Tensor& q,
                               const OptTensor& k, const OptTensor& q_weight,
                               const OptTensor& k_weight, const torch::Tensor& positions,
                               const torch::Tensor& freqs, const OptTensor& axes, double eps,
                               double weight_offset, bool interleaved, double scale,
                               const OptTensor& q_out, const OptTensor& k_out,
                               const OptTensor& dq_weight, const OptTensor& dk_weight,
                               const OptTensor& workspace) {
  fl_rotary_params p =
      rotary_params(dq, dk, first_axis(positions, axes), freqs, interleaved, scale);
  TORCH_CHECK(given(k) == given(dk), "k and dk are given both or not at all");
  const fl_norm_params n =
      norm_params(dq, dk, q_weight, k_weight, positions, axes, p.pairs, eps, weight_offset);
  const auto dev = dq.device();
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  fl_norm_grads d = {};
  view4(q, dq, "q", d.q_stride);
  TORCH_CHECK(q.sizes() == dq.sizes(), "q must have dq's shape");
  d.q = q.data_ptr();
  const torch::Tensor qo = given(q_out) ? *q_out : torch::empty_like(dq);
  view4(qo, dq, "q_out", p.q_out_stride);
  TORCH_CHECK(qo.sizes() == dq.sizes(), "q_out must have dq's shape");
  p.q_out = qo.data_ptr();
  torch::Tensor ko;
  if (given(dk)) {
    view4(*k, dq, "k", d.k_stride);
    TORCH_CHECK(k->sizes() == dk->sizes(), "k must have dk's shape");
    d.k = k->data_ptr();
    ko = given(k_out) ? *k_out : torch::empty_like(*dk);
    view4(ko, dq, "k_out", p.k_out_stride);
    TORCH_CHECK(ko.sizes() == dk->sizes(), "k_out must have dk's shape");
    p.k_out = ko.data_ptr();
  } else {
    TORCH_CHECK(!given(k_out), "k_out= needs dk");
  }
  TORCH_CHECK(given(q_weight) || !given(dq_weight), "dq_weight= needs q_weight");
  TORCH_CHECK(given(k_weight) || !given(dk_weight), "dk_weight= needs k_weight");
  torch::Tensor dqw, dkw, ws;
  if (given(q_weight)) {
    dqw = output(dq_weight, {p.head_dim}, torch::kFloat32, dev, "dq_weight");
    d.dq_weight = dqw.data_ptr<float>();
  }
  if (given(k_weight)) {
    dkw = output(dk_weight, {p.head_dim}, torch::kFloat32, dev, "dk_weight");
    d.dk_weight = dkw.data_ptr<float>();
  }
  const int64_t need = fl_attn_norm_rotary_workspace_bytes(&p);
  TORCH_CHECK(need >= 0, "FlashLite HIP error: ", fl_attn_last_error());
  if (given(q_weight) || given(k_weight)) ws = workspace_of(workspace, need, dq);
  ok(fl_attn_norm_rotary_bwd(&p, &n, &d, ws.defined() ? ws.data_ptr() : nullptr, need,
                             current_stream(dq)));
  auto or_none = [](const torch::Tensor& t) -> py::object {
    if (t.defined()) return py::cast(t);
    return py::none();
  };
  return py::make_tuple(qo, or_none(ko), or_none(dqw), or_none(dkw));
}

torch::Tensor norm_rotary_to_cache(const torch::Tensor& q, const torch::Tensor& k,
                                   const torch::Tensor& v, const OptTensor& q_weight,
                                   const OptTensor& k_weight, const torch::Tensor& positions,
                                   const torch::Tensor& slots, const torch::Tensor& freqs,
                                   const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                                   const OptTensor& axes, double eps, double weight_offset,
                                   bool interleaved, double scale, const OptTensor& out) {
  fl_rotary_params p =
      rotary_params(q, k, first_axis(positions, axes), freqs, interleaved, scale);
  const fl_norm_params n =
      norm_params(q, k, q_weight, k_weight, positions, axes, p.pairs, eps, weight_offset);
  const fl_cache_store c = cache_store(p, q, k, v, slots, k_cache, v_cache);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const torch::Tensor o = given(out) ? *out : torch::zeros_like(q);
  view4(o, q, "out", p.q_out_stride);
  TORCH_CHECK(o.sizes() == q.sizes(), "out must have q's shape");
  p.q_out = o.data_ptr();
  ok(fl_attn_norm_rotary_cache(&p, &n, &c, current_stream(q)));
  return o;
}

namespace {

fl_tree_params tree_sizes(const torch::Tensor& q, const torch::Tensor& k_cache) {
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  fl_tree_params p = {};
  p.dtype = serve_dtype(q);
  TORCH_CHECK(p.dtype == FL_DTYPE_F16 || p.dtype == FL_DTYPE_BF16,
              "All tensors must be FP16 (Half), or all BF16");
  view4(q, q, "q", p.q_stride);
  view4(k_cache, q, "k_cache", p.k_stride);
  TORCH_CHECK(k_cache.size(3) == q.size(3),
              "The caches must be [blocks, H_k, block_size, D] with q's D");
  p.batch = q.size(0);
  p.heads = q.size(1);
  p.drafts = q.size(2);
  p.head_dim = q.size(3);
  p.num_blocks = k_cache.size(0);
  p.kv_heads = k_cache.size(1);
  p.block_size = k_cache.size(2);
  return p;
}

}  // namespace

py::object forward_tree(const torch::Tensor& q, const torch::Tensor& k_cache,
                        const torch::Tensor& v_cache, const torch::Tensor& block_tables,
                        const torch::Tensor& lengths, const OptTensor& mask,
                        const OptTensor& counts, double sm_scale, const OptTensor& out,
                        bool return_lse, const OptTensor& lse, const OptTensor& workspace) {
  fl_tree_params p = tree_sizes(q, k_cache);
  const auto dev = q.device();
  view4(v_cache, q, "v_cache", p.v_stride);
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "v_cache must have k_cache's shape");
  check_int32(block_tables, dev, 2, "block_tables");
  TORCH_CHECK(block_tables.size(0) == p.batch &&
                  (block_tables.stride(1) == 1 || block_tables.size(1) <= 1),
              "block_tables must be [B, M] with unit-stride rows");
  p.block_tables = block_tables.data_ptr<int32_t>();
  p.table_stride = block_tables.stride(0);
  p.max_blocks = block_tables.size(1);
  p.lengths = requests(lengths, dev, p.batch, "lengths");
  p.counts = given(counts) ? requests(*counts, dev, p.batch, "counts") : nullptr;
  if (given(mask)) {
    const torch::Tensor& m = *mask;
    TORCH_CHECK(m.is_cuda() && m.device() == dev && m.scalar_type() == torch::kInt64,
                "mask must be int64 on the same device as the others");
    const int64_t words = (p.drafts + 63) / 64, d = m.dim();
    TORCH_CHECK((d == 2 || (d == 3 && m.size(0) == p.batch)) && m.size(d - 2) == p.drafts &&
                    m.size(d - 1) == words,
                "mask must be [B, n, W] or [n, W] with W = ceil(n / 64)");
    TORCH_CHECK((m.stride(d - 1) == 1 || words <= 1) &&
                    (m.stride(d - 2) == words || p.drafts <= 1),
                "mask must have contiguous rows");
    p.mask = m.data_ptr<int64_t>();
    p.mask_stride = d == 3 ? m.stride(0) : 0;
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  // Rows of drafts that are not there are not written: new outputs are zeros.
  const torch::Tensor o = given(out) ? *out
                          : p.counts ? torch::zeros_like(q)
                                     : torch::empty_like(q);
  view4(o, q, "out", p.o_stride);
  TORCH_CHECK(o.sizes() == q.sizes(), "out must have q's shape");
  torch::Tensor l;
  TORCH_CHECK(!given(lse) || return_lse, "lse= needs return_lse=True");
  if (return_lse) {
    l = output(lse, {p.batch, p.heads, p.drafts}, torch::kFloat32, dev, "lse");
    if (!given(lse) && p.counts) l.zero_();
    p.lse = l.data_ptr<float>();
  }
  p.q = q.data_ptr();
  p.k_cache = k_cache.data_ptr();
  p.v_cache = v_cache.data_ptr();
  p.o = o.data_ptr();
  p.sm_scale = sm_scale;
  const int64_t need = fl_attn_tree_workspace_bytes(&p);
  TORCH_CHECK(need >= 0, "FlashLite HIP error: ", fl_attn_last_error());
  torch::Tensor ws;
  if (need > 0) ws = workspace_of(workspace, need, q);
  ok(fl_attn_tree_fwd(&p, need > 0 ? ws.data_ptr() : nullptr, need, current_stream(q)));
  if (return_lse) return py::make_tuple(o, l);
  return py::cast(o);
}

// ---------------------------------------------------------------------------
// Attention over packed sequences (include/flashlite_attn.h).

namespace {

// A [1, heads, rows, D] view: strides {head, row}.
void view_packed(const torch::Tensor& t, const torch::Tensor& like, const char* name,
                 int64_t st[2]) {
  int64_t all[3];
  view4(t, like, name, all);
  TORCH_CHECK(t.size(0) == 1, name, " must be [1, heads, rows, D]: packed sequences are one batch");
  st[0] = all[1];
  st[1] = all[2];
}

fl_packed_params packed_params(const torch::Tensor& q, const torch::Tensor& k,
                               const torch::Tensor& v, const torch::Tensor& starts,
                               const OptTensor& key_starts, double sm_scale, bool is_causal) {
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  fl_packed_params p = {};
  p.dtype = serve_dtype(q);
  TORCH_CHECK(p.dtype == FL_DTYPE_F16 || p.dtype == FL_DTYPE_BF16,
              "All tensors must be FP16 (Half), or all BF16");
  view_packed(q, q, "q", p.q_stride);
  view_packed(k, q, "k", p.k_stride);
  view_packed(v, q, "v", p.v_stride);
  p.heads = q.size(1);
  p.rows = q.size(2);
  p.head_dim = q.size(3);
  p.kv_heads = k.size(1);
  p.key_rows = k.size(2);
  TORCH_CHECK(k.size(3) == p.head_dim && v.sizes() == k.sizes(),
              "k and v must be [1, H_k, T_k, D] with q's D");
  check_int32(starts, q.device(), 1, "starts");
  TORCH_CHECK(starts.size(0) >= 1 && starts.is_contiguous(),
              "starts must be contiguous, [sequences + 1]");
  p.sequences = starts.size(0) - 1;
  p.starts = starts.data_ptr<int32_t>();
  if (given(key_starts)) {
    check_int32(*key_starts, q.device(), 1, "key_starts");
    TORCH_CHECK(key_starts->sizes() == starts.sizes() && key_starts->is_contiguous(),
                "key_starts must be contiguous, with as many entries as starts");
    p.key_starts = key_starts->data_ptr<int32_t>();
  } else {
    TORCH_CHECK(p.key_rows == p.rows, "k must have q's rows without key_starts");
  }
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  for (int i = 0; i < 2; ++i) p.o_stride[i] = p.q_stride[i];
  p.sm_scale = sm_scale;
  p.causal = is_causal ? 1 : 0;
  return p;
}

}  // namespace

py::object forward_packed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                          const torch::Tensor& starts, const OptTensor& key_starts,
                          double sm_scale, bool is_causal, const OptTensor& out, bool return_lse,
                          const OptTensor& lse) {
  fl_packed_params p = packed_params(q, k, v, starts, key_starts, sm_scale, is_causal);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  // Rows of no sequence are not written: new outputs are zeros.
  const torch::Tensor o = given(out) ? *out : torch::zeros_like(q);
  view_packed(o, q, "out", p.o_stride);
  TORCH_CHECK(o.sizes() == q.sizes(), "out must have q's shape");
  p.o = o.data_ptr();
  torch::Tensor l;
  TORCH_CHECK(!given(lse) || return_lse, "lse= needs return_lse=True");
  if (return_lse) {
    l = output(lse, {1, p.heads, p.rows}, torch::kFloat32, q.device(), "lse");
    if (!given(lse)) l.zero_();
    p.lse = l.data_ptr<float>();
  }
  ok(fl_attn_packed_fwd(&p, current_stream(q)));
  if (return_lse) return py::make_tuple(o, l);
  return py::cast(o);
}

py::tuple backward_packed(const torch::Tensor& dout, const torch::Tensor& q, const torch::Tensor& k,
                          const torch::Tensor& v, const torch::Tensor& out,
                          const torch::Tensor& lse, const torch::Tensor& starts,
                          const OptTensor& key_starts, double sm_scale, bool is_causal,
                          const OptTensor& dq, const OptTensor& dk, const OptTensor& dv,
                          const OptTensor& workspace) {
  fl_packed_params p = packed_params(q, k, v, starts, key_starts, sm_scale, is_causal);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  fl_packed_grads d = {};
  view_packed(out, q, "out", p.o_stride);
  view_packed(dout, q, "dout", d.dout_stride);
  TORCH_CHECK(out.sizes() == q.sizes() && dout.sizes() == q.sizes(),
              "out and dout must have q's shape");
  p.o = out.data_ptr();
  d.dout = dout.data_ptr();
  p.lse = output(lse, {1, p.heads, p.rows}, torch::kFloat32, q.device(), "lse").data_ptr<float>();
  auto gradient = [&](const OptTensor& t, const torch::Tensor& like, const char* name,
                      int64_t st[2]) {
    const torch::Tensor x = given(t) ? *t : torch::zeros_like(like);
    view_packed(x, q, name, st);
    TORCH_CHECK(x.sizes() == like.sizes(), name, " must have its input's shape");
    return x;
  };
  const torch::Tensor gq = gradient(dq, q, "dq", d.dq_stride);
  const torch::Tensor gk = gradient(dk, k, "dk", d.dk_stride);
  const torch::Tensor gv = gradient(dv, v, "dv", d.dv_stride);
  d.dq = gq.data_ptr();
  d.dk = gk.data_ptr();
  d.dv = gv.data_ptr();
  const int64_t need = fl_attn_packed_bwd_workspace_bytes(&p);
  TORCH_CHECK(need >= 0, "FlashLite HIP error: ", fl_attn_last_error());
  torch::Tensor ws;
  if (need > 0) ws = workspace_of(workspace, need, q);
  ok(fl_attn_packed_bwd(&p, &d, need > 0 ? ws.data_ptr() : nullptr, need, current_stream(q)));
  return py::make_tuple(gq, gk, gv);
}

}  // namespace flash_attn

PYBIND11_MODULE(flash_attn_wmma, m) {
  m.doc() = "FlashAttention-2 forward for AMD Instinct MI355X (gfx950): MFMA + LDS HIP kernels";

  m.def("forward_naive", &flash_attn::flash_attn_forward_naive,
        "Naive attention forward (HIP baseline, one work-group per query row)", py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("sm_scale") = 0.0, py::arg("is_causal") = false);

  m.def("forward_flash2", &flash_attn::flash_attn_forward_flash2,
        "FlashAttention-2 forward (gfx950 MFMA)", py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("sm_scale") = 0.0, py::arg("is_causal") = false, py::arg("out") = py::none());

  m.def("forward_flash2_ex", &flash_attn::flash_attn_forward_flash2_ex,
        "FlashAttention-2 forward on strided [B, H, N, D] views (fp16 or bf16, D 64 or 128), "
        "N_k != N_q (bottom-right causal), optional log-sum-exp.  Few query rows over many keys "
        "run as key chunks through `workspace` (splitkv_workspace_bytes bytes on q's device); "
        "calls that may overlap on the GPU must not share one.  Without it bf16 and head_dim 128 "
        "calls that are given their outputs run one pass and allocate nothing",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("sm_scale") = 0.0,
        py::arg("is_causal") = false, py::arg("out") = py::none(), py::arg("return_lse") = false,
        py::arg("num_splits") = 0, py::arg("workspace") = py::none(), py::arg("lse") = py::none());

  m.def("splitkv_workspace_bytes",
        [](torch::Tensor q, torch::Tensor k, bool is_causal, int64_t num_splits) {
          fl_attn_params_ex p;
          p.base = fl_attn_params{nullptr, nullptr, nullptr, nullptr, q.size(0), q.size(1),
                                  q.size(2), k.size(2), q.size(3), 0.0, is_causal ? 1 : 0};
          const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)};
          const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)};
          for (int d = 0; d < 3; ++d) {
            p.q_stride[d] = p.o_stride[d] = qs[d];
            p.k_stride[d] = p.v_stride[d] = ks[d];
          }
          p.lse = nullptr;
          if (num_splits == 1) return (int64_t)0;
          const bool bf16 = q.scalar_type() == torch::kBFloat16;
          if (q.scalar_type() != torch::kHalf || q.size(3) != 64) {
            // bf16 and head_dim 128 split by the library's choice only; what
            // forward_flash2_ex will refuse needs no workspace
            if (num_splits != 0 || (!bf16 && q.scalar_type() != torch::kHalf)) return (int64_t)0;
            const int64_t w = fl_attn_workspace_bytes(&p, bf16 ? FL_DTYPE_BF16 : FL_DTYPE_F16);
            return w > 0 ? w : (int64_t)0;
          }
          const int64_t b = fl_attn_splitkv_workspace_bytes(&p, (int32_t)num_splits);
          TORCH_CHECK(b >= 0, "FlashLite HIP error: ", fl_attn_last_error());
          return b;
        },
        "Workspace bytes forward_flash2_ex needs for these q / k shapes and num_splits "
        "(0 when it runs one pass)",
        py::arg("q"), py::arg("k"), py::arg("is_causal") = false, py::arg("num_splits") = 0);

  m.def("plan_cache", &flash_attn::plan_cache,
        "Blocks, slots and positions of a step's new tokens in a paged cache, from the requests' "
        "lengths: returns (positions [B, width] int32, slots [B, width] int64, info [B, 4] int32) "
        "and updates block_tables, held (or held_out) and free_state (or state_out). counts < 0 "
        "ends a request: its blocks go back to the ring free_blocks",
        py::arg("lengths"), py::arg("counts"), py::arg("block_tables"), py::arg("held"),
        py::arg("free_blocks"), py::arg("free_state"), py::arg("block_size"), py::arg("width"),
        py::arg("held_out") = py::none(), py::arg("state_out") = py::none(),
        py::arg("positions") = py::none(), py::arg("slots") = py::none(),
        py::arg("info") = py::none());

  m.def("plan_tree", &flash_attn::plan_tree,
        "Ancestors' bits [B, n, ceil(n / 64)] int64 and positions [B, n] int32 of drafted tokens "
        "from each draft's parent (an earlier draft; anything else: the request's last token)",
        py::arg("parents"), py::arg("lengths"), py::arg("counts") = py::none(),
        py::arg("mask") = py::none(), py::arg("positions") = py::none());

  m.def("forward_rotary", &flash_attn::forward_rotary,
        "Rotary positions of q and k (or None) [B, H, N, D] views, D 64 or 128, fp16, bf16 or "
        "fp32: pairs {j, j + len(freqs)}, or {2j, 2j + 1} with interleaved, turn by "
        "positions * freqs[j] (float64 radians) and are multiplied by scale; the outputs may be "
        "the inputs. Not recorded by autograd: the gradient is backward_rotary",
        py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("freqs"),
        py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("q_out") = py::none(),
        py::arg("k_out") = py::none());

  m.def("backward_rotary", &flash_attn::backward_rotary,
        "The gradient of forward_rotary: the same call on the outputs' gradients, the angles "
        "negated. Not recorded by autograd itself",
        py::arg("dq"), py::arg("dk"), py::arg("positions"), py::arg("freqs"),
        py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("q_out") = py::none(),
        py::arg("k_out") = py::none());

  m.def("rotary_to_cache", &flash_attn::rotary_to_cache,
        "Rotates q into out, and stores rotated k and v in row slots[b][i] of the paged caches "
        "[blocks, H_k, block_size, D]; tokens with a negative slot are passed over. Slots must "
        "differ",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("positions"), py::arg("slots"),
        py::arg("freqs"), py::arg("k_cache"), py::arg("v_cache"), py::arg("interleaved") = false,
        py::arg("scale") = 1.0, py::arg("out") = py::none());

  m.def("forward_tree", &flash_attn::forward_tree,
        "Attention of drafted tokens q [B, H, n, D] over a paged cache [blocks, H_k, block_size, "
        "D]: draft i sees its request's lengths[b] tokens and the drafts in its mask (None: a "
        "chain; n = 1 is a decode step), whose keys and values are in the cache behind them. "
        "Returns out, or (out, lse). workspace: tree_workspace_bytes(q, k_cache) bytes, or one "
        "from the caching allocator; calls that may overlap on the GPU must not share one",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_tables"),
        py::arg("lengths"), py::arg("mask") = py::none(), py::arg("counts") = py::none(),
        py::arg("sm_scale") = 0.0, py::arg("out") = py::none(), py::arg("return_lse") = false,
        py::arg("lse") = py::none(), py::arg("workspace") = py::none());

  m.def("tree_workspace_bytes",
        [](const torch::Tensor& q, const torch::Tensor& k_cache) {
          fl_tree_params p = flash_attn::tree_sizes(q, k_cache);
          for (int i = 0; i < 3; ++i) {
            p.o_stride[i] = p.q_stride[i];
            p.v_stride[i] = p.k_stride[i];
          }
          p.max_blocks = 1;
          p.table_stride = 1;
          const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
          const int64_t b = fl_attn_tree_workspace_bytes(&p);
          TORCH_CHECK(b >= 0, "FlashLite HIP error: ", fl_attn_last_error());
          return b;
        },
        "Workspace bytes of forward_tree for these q and k_cache (0: none is used)", py::arg("q"),
        py::arg("k_cache"));

  m.def("forward_norm_rotary", &flash_attn::forward_norm_rotary,
        "Norms of q and k (or None) [B, H, N, D] views for each head and rotary positions in one "
        "pass: x / sqrt(mean(x x) + eps) * (weight + weight_offset), then the rotation of "
        "forward_rotary. A weight [D] (FP32 or of q's dtype) of None leaves its tensor without a "
        "norm. axes: int32, the axis of each pair, with positions [A, B, N] (or [A, N]). The "
        "outputs may be the inputs. Not recorded by autograd: the gradient is "
        "backward_norm_rotary",
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("positions"),
        py::arg("freqs"), py::arg("axes") = py::none(), py::arg("eps") = 1e-6,
        py::arg("weight_offset") = 0.0, py::arg("interleaved") = false, py::arg("scale") = 1.0,
        py::arg("q_out") = py::none(), py::arg("k_out") = py::none());

  m.def("backward_norm_rotary", &flash_attn::backward_norm_rotary,
        "The gradients of forward_norm_rotary from those of its outputs, dq and dk, and its inputs "
        "q and k: returns (dq, dk, dq_weight, dk_weight), the weights' in FP32, None for what is "
        "not there. q_out and k_out may be dq and dk. workspace: norm_rotary_workspace_bytes(q, k) "
        "bytes, or one from the caching allocator; calls that may overlap on the GPU must not "
        "share one. Not recorded by autograd itself",
        py::arg("dq"), py::arg("dk"), py::arg("q"), py::arg("k"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("positions"), py::arg("freqs"), py::arg("axes") = py::none(),
        py::arg("eps") = 1e-6, py::arg("weight_offset") = 0.0, py::arg("interleaved") = false,
        py::arg("scale") = 1.0, py::arg("q_out") = py::none(), py::arg("k_out") = py::none(),
        py::arg("dq_weight") = py::none(), py::arg("dk_weight") = py::none(),
        py::arg("workspace") = py::none());

  m.def("norm_rotary_workspace_bytes",
        [](const torch::Tensor& q, const std::optional<torch::Tensor>& k) {
          (void)k;
          TORCH_CHECK(q.dim() == 4, "q must be 4D");
          fl_rotary_params p = {};
          p.head_dim = q.size(3);
          const int64_t b = fl_attn_norm_rotary_workspace_bytes(&p);
          TORCH_CHECK(b >= 0, "FlashLite HIP error: ", fl_attn_last_error());
          return b;
        },
        "Workspace bytes of backward_norm_rotary for these q and k", py::arg("q"),
        py::arg("k") = py::none());

  m.def("norm_rotary_to_cache", &flash_attn::norm_rotary_to_cache,
        "forward_norm_rotary for a step's tokens: q goes into out, and k with v into row "
        "slots[b][i] of the paged caches, as rotary_to_cache stores them",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("q_weight"), py::arg("k_weight"),
        py::arg("positions"), py::arg("slots"), py::arg("freqs"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("axes") = py::none(), py::arg("eps") = 1e-6,
        py::arg("weight_offset") = 0.0, py::arg("interleaved") = false, py::arg("scale") = 1.0,
        py::arg("out") = py::none());

  m.def("forward_packed", &flash_attn::forward_packed,
        "Attention over packed sequences of different lengths: q [1, H, T, D], k and v [1, H_k, "
        "T_k, D] views (FP16 or BF16, D 64 or 128), sequence i the rows starts[i] .. starts[i + 1] "
        "- 1 of q and key_starts[i] .. (None: the same) of k and v; starts int32 [sequences + 1]. "
        "Grouped heads; causal: the last query sees all of its sequence's keys. Rows of no "
        "sequence are left as they were. Returns out, or (out, lse [1, H, T]). Not recorded by "
        "autograd: the gradient is backward_packed",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("starts"),
        py::arg("key_starts") = py::none(), py::arg("sm_scale") = 0.0,
        py::arg("is_causal") = false, py::arg("out") = py::none(), py::arg("return_lse") = false,
        py::arg("lse") = py::none());

  m.def("backward_packed", &flash_attn::backward_packed,
        "The gradients (dq, dk, dv) of forward_packed from dout and its inputs, out and lse; the "
        "same inputs give the same bits. workspace: packed_workspace_bytes(q, k, starts) bytes, or "
        "one from the caching allocator; calls that may overlap on the GPU must not share one. Not "
        "recorded by autograd itself",
        py::arg("dout"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("out"), py::arg("lse"),
        py::arg("starts"), py::arg("key_starts") = py::none(), py::arg("sm_scale") = 0.0,
        py::arg("is_causal") = false, py::arg("dq") = py::none(), py::arg("dk") = py::none(),
        py::arg("dv") = py::none(), py::arg("workspace") = py::none());

  m.def("packed_workspace_bytes",
        [](const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& starts) {
          const fl_packed_params p =
              flash_attn::packed_params(q, k, k, starts, starts, 0.0, false);
          const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
          const int64_t b = fl_attn_packed_bwd_workspace_bytes(&p);
          TORCH_CHECK(b >= 0, "FlashLite HIP error: ", fl_attn_last_error());
          return b;
        },
        "Workspace bytes of backward_packed for these q, k and starts", py::arg("q"), py::arg("k"),
        py::arg("starts"));
}
