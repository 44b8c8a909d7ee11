// Python bindings of the serving operators over a paged key / value cache.  Arguments are checked here (ValueError); what only the
// device knows (lengths, page ids) is bounds-checked by the kernels.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "api_paged.h"
#include "binding.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, " (", rc < 1000 ? cudaGetErrorString((cudaError_t)rc) : "driver", ")");
}

int type_of(const Tensor& x, const char* name) {
  switch (x.scalar_type()) {
    case at::kFloat: return LBI_F32;
    case at::kBFloat16: return LBI_BF16;
    case at::kHalf: return LBI_F16;
    default: TORCH_CHECK_VALUE(false, name, " must be fp32, bf16 or fp16");
  }
}

bool given(const OptTensor& x) { return x.has_value() && x->defined(); }

void check_int32(const Tensor& x, const Tensor& like, int64_t dims, const char* name) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kInt && x.dim() == dims && x.device() == like.device(), name, " must be an int32 tensor of ", dims,
                    " dimension(s) on the pages' device");
  TORCH_CHECK_VALUE(x.numel() == 0 || x.size(-1) <= 1 || x.stride(-1) == 1, name, " must be contiguous along its last dimension");
}

// Checks the cache and the batch and fills the geometry; `rows` new tokens.
lbi_paged_batch paged_batch(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& table,
                            const Tensor& context, const OptTensor& cu, int64_t rows) {
  TORCH_CHECK_VALUE(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && k.sizes() == v.sizes() &&
                        k.scalar_type() == v.scalar_type() && k.device() == v.device(),
                    "k and v pages must be contiguous [num_pages, kv_heads, page_size, head_dim] tensors of one type on one device");
  lbi_paged_batch p{};
  const int64_t page = k.size(2);
  TORCH_CHECK_VALUE(page >= 8 && page <= 128 && (page & (page - 1)) == 0, "page_size must be a power of two in 8 .. 128, got ", page);
  TORCH_CHECK_VALUE(k.size(0) > 0 && k.size(1) > 0, "the pages hold nothing");
  TORCH_CHECK_VALUE(k.size(0) * k.size(1) * page < (1ll << 31), "the pages have 2^31 slots or more");
  TORCH_CHECK_VALUE((uintptr_t)k.data_ptr() % 16 == 0 && (uintptr_t)v.data_ptr() % 16 == 0, "the pages must start on a 16-byte boundary");
  if (k.scalar_type() == at::kFloat8_e4m3fn) {
    TORCH_CHECK_VALUE(given(k_scale) && given(v_scale), "e4m3 pages need k_scale and v_scale");
    for (const Tensor& s : {*k_scale, *v_scale})
      TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.is_contiguous() && s.device() == k.device() && s.dim() == 3 &&
                            s.size(0) == k.size(0) && s.size(1) == k.size(1) && s.size(2) == page,
                        "scales must be contiguous fp32 [num_pages, kv_heads, page_size] tensors");
    p.k_scale = k_scale->data_ptr<float>();
    p.v_scale = v_scale->data_ptr<float>();
    p.cache_type = LBI_E4M3;
  } else {
    TORCH_CHECK_VALUE(!given(k_scale) && !given(v_scale), "only e4m3 pages have scales");
    p.cache_type = type_of(k, "pages");
  }
  check_int32(table, k, 2, "page_table");
  check_int32(context, k, 1, "context_lens");
  p.batch = (int)context.size(0);
  TORCH_CHECK_VALUE(table.size(0) == p.batch, "page_table has ", table.size(0), " rows for ", p.batch, " context lengths");
  // room for a tile behind the last position: the kernels count positions in 32 bits
  TORCH_CHECK_VALUE(table.size(1) * page < (1ll << 31) - 65536, "2^31 - 65536 positions in the page table or more");
  TORCH_CHECK_VALUE(rows < (1ll << 31), "2^31 rows or more");
  if (given(cu)) {
    check_int32(*cu, k, 1, "cu_seqlens");
    TORCH_CHECK_VALUE(cu->size(0) == p.batch + 1, "cu_seqlens must have one entry more than context_lens");
    p.cu = cu->data_ptr<int>();
  } else {
    TORCH_CHECK_VALUE(p.batch == 0 ? rows == 0 : rows % p.batch == 0, "without cu_seqlens the rows must divide evenly among the sequences");
  }
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.table = table.data_ptr<int>();
  p.context = context.data_ptr<int>();
  p.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  p.num_pages = (int)k.size(0);
  p.kv_heads = (int)k.size(1);
  p.page_size = (int)page;
  p.head_dim = (int)k.size(3);
  p.table_width = (int)table.size(1);
  p.rows = (int)rows;
  p.status = status_word(k).data_ptr<int>();
  return p;
}

// Inner dimension contiguous, rows and base on 16-byte boundaries: what the kernels' wide loads need.
Tensor aligned_rows(const Tensor& x) {
  const int64_t item = x.element_size();
  if (x.stride(-1) == 1 && (x.size(0) <= 1 || (x.stride(0) * item) % 16 == 0) && (uintptr_t)x.data_ptr() % 16 == 0) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

Tensor output(const OptTensor& out, at::IntArrayRef sizes, const Tensor& like, at::ScalarType type, bool nobody = false) {
  if (!given(out)) {
    Tensor made = at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);   // without the dispatcher: a decode loop waits for the host
    return nobody ? made.zero_() : made;
  }
  TORCH_CHECK_VALUE(out->sizes() == sizes && out->scalar_type() == type && out->device() == like.device() && out->is_contiguous() &&
                        (uintptr_t)out->data_ptr() % 16 == 0,
                    "out must be a contiguous tensor of the result's shape and type on its device");
  return *out;
}

void check_cache_type(const Tensor& x, const Tensor& k) {
  TORCH_CHECK_VALUE(x.device() == k.device(), "the rows and the pages must be on one device");
  TORCH_CHECK_VALUE(k.scalar_type() == x.scalar_type() || k.scalar_type() == at::kFloat8_e4m3fn, "the pages hold ", k.scalar_type(),
                    ": they must hold the rows' type (", x.scalar_type(), ") or e4m3");
}

Tensor kv_append(const Tensor& qkv_in, const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& table,
                 const Tensor& context, int64_t heads, const OptTensor& cu, const OptTensor& cos_tab, const OptTensor& sin_tab, bool interleaved,
                 const OptTensor& out) {
  TORCH_CHECK_VALUE(qkv_in.is_cuda() && qkv_in.dim() == 2, "qkv must be a CUDA tensor [rows, (heads + 2 kv_heads) * head_dim]");
  check_cache_type(qkv_in, k);
  c10::cuda::CUDAGuard guard(k.device());
  const lbi_paged_batch p = paged_batch(k, v, k_scale, v_scale, table, context, cu, qkv_in.size(0));
  TORCH_CHECK_VALUE(heads > 0 && qkv_in.size(1) == (heads + 2 * p.kv_heads) * p.head_dim, "qkv has ", qkv_in.size(1), " columns for ", heads, " + 2 x ",
                    p.kv_heads, " heads of ", p.head_dim);
  const float *cp = nullptr, *sp = nullptr;
  int64_t rope_rows = 0;
  TORCH_CHECK_VALUE(given(cos_tab) == given(sin_tab), "rope needs both tables");
  if (given(cos_tab)) {
    for (const Tensor& t : {*cos_tab, *sin_tab})
      TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(1) == p.head_dim / 2 && t.is_contiguous() && t.device() == k.device() &&
                            (uintptr_t)t.data_ptr() % 16 == 0 && t.size(0) == cos_tab->size(0),
                        "rotary tables must be contiguous fp32 [positions, head_dim / 2] tensors on the pages' device");
    cp = cos_tab->data_ptr<float>();
    sp = sin_tab->data_ptr<float>();
    rope_rows = cos_tab->size(0);
  }
  const Tensor qkv = aligned_rows(qkv_in);
  Tensor q = output(out, {qkv.size(0), heads, (int64_t)p.head_dim}, qkv, qkv.scalar_type());
  check(lbi_kv_append(&p, qkv.data_ptr(), qkv.stride(0), q.data_ptr(), type_of(qkv, "qkv"), (int)heads, cp, sp, rope_rows, interleaved ? 1 : 0,
                      given(out) ? 0 : 1, cur_stream()),
        "kv_append");
  return q;
}

std::tuple<Tensor, Tensor> kv_gather(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& table,
                                     const Tensor& context, int64_t max_len, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(max_len >= 0, "max_len must not be negative");
  c10::cuda::CUDAGuard guard(k.device());
  const lbi_paged_batch p = paged_batch(k, v, k_scale, v_scale, table, context, c10::nullopt, 0);
  Tensor ko = output(c10::nullopt, {p.batch, p.kv_heads, max_len, p.head_dim}, k, dtype);
  Tensor vo = output(c10::nullopt, {p.batch, p.kv_heads, max_len, p.head_dim}, k, dtype);
  const int type = type_of(ko, "dtype");
  TORCH_CHECK_VALUE(p.cache_type == LBI_E4M3 || p.cache_type == type, "pages that are not e4m3 are read back in their own type");
  check(lbi_kv_gather(&p, ko.data_ptr(), vo.data_ptr(), max_len, type, cur_stream()), "kv_gather");
  return {ko, vo};
}

Tensor paged_attention(const Tensor& q_in, const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& table,
                       const Tensor& context, double scale, const OptTensor& cu, int64_t max_context, const OptTensor& out) {
  TORCH_CHECK_VALUE(max_context >= 0, "max_context must not be negative");
  TORCH_CHECK_VALUE(q_in.is_cuda() && q_in.dim() == 3, "q must be a CUDA tensor [rows, heads, head_dim]");
  check_cache_type(q_in, k);
  c10::cuda::CUDAGuard guard(k.device());
  const lbi_paged_batch p = paged_batch(k, v, k_scale, v_scale, table, context, cu, q_in.size(0));
  const int64_t heads = q_in.size(1);
  TORCH_CHECK_VALUE(heads > 0 && heads % p.kv_heads == 0 && q_in.size(2) == p.head_dim, "q has ", heads, " heads of ", q_in.size(2), ": pages have ",
                    p.kv_heads, " of ", p.head_dim);
  TORCH_CHECK_VALUE(q_in.size(0) * heads < (1ll << 31), "2^31 rows times heads or more");
  const bool packed = q_in.stride(2) == 1 && (heads == 1 || q_in.stride(1) == p.head_dim);
  const Tensor q = aligned_rows(packed ? q_in : q_in.contiguous());
  Tensor o = output(out, q.sizes(), q, q.scalar_type(), p.batch == 0);
  const int type = type_of(q, "q");
  const int sm_count = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const lbi_attention_plan plan = lbi_paged_attention_plan(&p, type, (int)heads, (float)scale, max_context, sm_count);
  Tensor parts;   // results of the parts of a long context, then the logarithms of their sums
  const int64_t part_rows = q.size(0) * heads * plan.splits;
  if (plan.splits > 1) parts = at::detail::empty_cuda({part_rows * (p.head_dim + 1)}, at::kFloat, q.device(), c10::nullopt);
  float* part_o = plan.splits > 1 ? parts.data_ptr<float>() : nullptr;
  check(lbi_paged_attention(&p, q.data_ptr(), q.size(0) > 1 ? q.stride(0) : heads * p.head_dim, o.data_ptr(), part_o,
                            part_o ? part_o + part_rows * p.head_dim : nullptr, plan, type, (int)heads, (float)scale, given(out) ? 0 : 1, sm_count, cur_stream()),
        "paged_attention");
  return o;
}

// A penalty is a number or one fp32 entry per row: fills whichever it is.
void penalty(const py::object& x, const Tensor& like, const char* name, const float** row, float* number) {
  if (!THPVariable_Check(x.ptr())) {
    *number = (float)x.cast<double>();
    return;
  }
  const Tensor& t = THPVariable_Unpack(x.ptr());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == like.size(0) && t.is_contiguous() && t.device() == like.device(),
                    name, " must be a number or a contiguous fp32 tensor with one entry per row");
  *row = t.data_ptr<float>();
}

Tensor adjust_logits(const Tensor& logits, const Tensor& tokens, const OptTensor& lengths, const OptTensor& prompt_lengths, const py::object& repetition,
                     const py::object& presence, const py::object& frequency, const OptTensor& bias, const OptTensor& allowed, const OptTensor& out) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
                    "logits must be a CUDA tensor [batch, vocab], contiguous along the vocabulary");
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t batch = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK_VALUE(vocab < (1ll << 31) - 65536 && batch < (1ll << 31), "2^31 entries or rows or more");
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong && tokens.dim() == 2 && tokens.size(0) == batch && tokens.device() == logits.device() &&
                        (tokens.size(1) <= 1 || tokens.stride(1) == 1) && tokens.size(1) < (1ll << 31) - 65536,   // the kernel's steps stay whole numbers
                    "tokens must be an int64 tensor [batch, history], contiguous along the history, of fewer than 2^31 - 65536 entries a row");
  lbi_logit_rules p{};
  p.type = type_of(logits, "logits");
  p.batch = (int)batch;
  p.vocab = (int)vocab;
  p.history = (int)tokens.size(1);
  p.logits = logits.data_ptr();
  p.logits_stride = batch > 1 ? logits.stride(0) : vocab;
  p.tokens = tokens.data_ptr<int64_t>();
  p.tokens_stride = batch > 1 ? tokens.stride(0) : tokens.size(1);
  for (const auto& x : {std::make_pair(&lengths, &p.lengths), std::make_pair(&prompt_lengths, &p.prompt_lengths)}) {
    if (!given(*x.first)) continue;
    check_int32(**x.first, logits, 1, "lengths");
    TORCH_CHECK_VALUE((*x.first)->size(0) == batch, "lengths must have one entry per row");
    *x.second = (*x.first)->data_ptr<int>();
  }
  penalty(repetition, logits, "repetition", &p.repetition_row, &p.repetition);
  penalty(presence, logits, "presence", &p.presence_row, &p.presence);
  penalty(frequency, logits, "frequency", &p.frequency_row, &p.frequency);
  TORCH_CHECK_VALUE(p.repetition_row || p.repetition > 0, "repetition must be positive");
  if (given(bias)) {
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->device() == logits.device() && bias->dim() >= 1 && bias->size(-1) == vocab &&
                          (bias->dim() == 1 || (bias->dim() == 2 && bias->size(0) == batch)) && (vocab <= 1 || bias->stride(-1) == 1),
                      "bias must be an fp32 tensor [vocab] or [batch, vocab]");
    p.bias = bias->data_ptr<float>();
    p.bias_stride = bias->dim() == 2 && batch > 1 ? bias->stride(0) : 0;
  }
  if (given(allowed)) {
    const int64_t words = (vocab + 31) / 32;
    TORCH_CHECK_VALUE(allowed->scalar_type() == at::kInt && allowed->device() == logits.device() && allowed->dim() >= 1 && allowed->size(-1) == words &&
                          (allowed->dim() == 1 || (allowed->dim() == 2 && allowed->size(0) == batch)) && (words <= 1 || allowed->stride(-1) == 1),
                      "allowed must be an int32 tensor [ceil(vocab / 32)] or [batch, ceil(vocab / 32)]");
    p.allowed = allowed->data_ptr<int>();
    p.allowed_stride = allowed->dim() == 2 && batch > 1 ? allowed->stride(0) : 0;
  }
  Tensor o = output(out, logits.sizes(), logits, at::kFloat);
  p.out = o.data_ptr<float>();
  p.out_stride = vocab;
  check(lbi_adjust_logits(&p, at::cuda::getCurrentDeviceProperties()->multiProcessorCount, cur_stream()), "adjust_logits");
  return o;
}

}  // namespace

void bind_paged(pybind11::module& m) {
  m.def("kv_append", &kv_append);
  m.def("kv_gather", &kv_gather);
  m.def("paged_attention", &paged_attention);
  m.def("adjust_logits", &adjust_logits);
}
