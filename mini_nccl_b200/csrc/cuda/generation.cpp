// Torch entry points of the generation operators: checks of the tensors, their
// workspaces, and the launches (cache.cu, sampling.cu, prefix_attention.cu).
#include "generation.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

namespace mnb {

namespace {

constexpr double kLog2e = 1.4426950408889634;

thread_local int64_t launched = 0;  // kernels of the last call

void check_int32(const torch::Tensor& t, int64_t dim, const torch::Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == dim &&
                        (t.numel() == 0 || t.size(dim - 1) == 1 || t.stride(dim - 1) == 1),
                    what, ": a ", dim, "-d int32 tensor on ", like.device(), " with its last axis contiguous");
  TORCH_CHECK_VALUE(t.numel() < (1ll << 31), what, ": too many entries");
}

void check_status_word(const torch::Tensor& status) {
  TORCH_CHECK(status.is_cuda() && status.scalar_type() == at::kInt && status.numel() >= 3, "status: int32 on the device");
}

// A device's status: word 0 is a pipeline wait that ran out, which makes every other wait give up too; word 2 a request
// that a kernel left out, which must not.
int* waits_of(const torch::Tensor& status) { return status.data_ptr<int>(); }
int* errors_of(const torch::Tensor& status) { return status.data_ptr<int>() + 2; }

// 16-byte accesses along the last axis work at every index.
bool rows_aligned(const torch::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) * t.element_size() % 16 == 0);
  return ok;
}

__nv_bfloat16* bf16(const torch::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }
uint8_t* bytes(const torch::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

using Scales = c10::optional<torch::Tensor>;

// The kind of a cache's pages; those in 8 bits come with a scale for each page and kv head.
prefix::Codes codes_of(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const Scales& k_scales, const Scales& v_scales) {
  const auto type = k_pages.scalar_type();
  const auto codes = type == at::kChar ? prefix::kInt8 : type == at::kFloat8_e4m3fn ? prefix::kE4m3 : prefix::kNoCodes;
  TORCH_CHECK_VALUE((codes || type == at::kBFloat16) && v_pages.scalar_type() == type && k_pages.is_cuda() && k_pages.dim() == 4 &&
                        v_pages.sizes() == k_pages.sizes() && v_pages.strides() == k_pages.strides() && v_pages.device() == k_pages.device(),
                    "k_pages and v_pages: bf16, int8 or float8_e4m3fn CUDA tensors [num_pages, page_size, kv_heads, head_dim] of one layout");
  TORCH_CHECK_VALUE(codes ? k_scales && v_scales : !k_scales && !v_scales,
                    "k_scales and v_scales: needed with pages of int8 or float8_e4m3fn, and only with them");
  if (codes)
    for (const auto* s : {&*k_scales, &*v_scales})
      TORCH_CHECK_VALUE(s->device() == k_pages.device() && s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == k_pages.size(0) &&
                            s->size(1) == k_pages.size(2) && s->strides() == k_scales->strides(),
                        "k_scales and v_scales: fp32 tensors [num_pages, kv_heads] of one layout, on the pages' device");
  return codes;
}

cache::Pool pool_of(const torch::Tensor& kv, const Scales& scales) {
  TORCH_CHECK_VALUE(kv.is_cuda() && kv.dim() >= 4 && kv.is_contiguous(),
                    "kv: a contiguous CUDA tensor [..., num_pages, page_size, kv_heads, head_dim]");
  TORCH_CHECK_VALUE(kv.numel() > 0, "kv: an empty pool");
  const int64_t d = kv.dim();
  const int64_t token = kv.size(d - 1) * kv.size(d - 2) * kv.element_size();
  const int64_t page = token * kv.size(d - 3), pages = kv.size(d - 4);
  TORCH_CHECK_VALUE(token % 16 == 0 && reinterpret_cast<uintptr_t>(kv.data_ptr()) % 16 == 0,
                    "kv: a token's keys must be a multiple of 16 bytes, 16-byte aligned (got ", token, " bytes)");
  TORCH_CHECK_VALUE(page / 16 < (1 << 30) && pages < (1 << 29), "kv: pages too large");
  cache::Pool p;
  p.base = kv.data_ptr();
  p.plane_chunks = pages * (page / 16);
  p.page_chunks = static_cast<int>(page / 16);
  p.token_chunks = static_cast<int>(token / 16);
  p.planes = static_cast<int>(kv.numel() * kv.element_size() / (page * pages));
  p.pages = static_cast<int>(pages);
  p.page_size = static_cast<int>(kv.size(d - 3));
  p.scales = nullptr;
  p.heads = 0;
  if (scales) {
    bool fits = scales->device() == kv.device() && scales->scalar_type() == at::kFloat && scales->is_contiguous() && scales->dim() == d - 2;
    for (int64_t i = 0; fits && i < d - 2; ++i) fits = scales->size(i) == kv.size(i < d - 3 ? i : d - 2);
    TORCH_CHECK_VALUE(fits, "scales: a contiguous fp32 tensor [..., num_pages, kv_heads] with the leading axes of kv");
    p.scales = scales->data_ptr<float>();
    p.heads = static_cast<int>(kv.size(d - 2));
  }
  return p;
}

cache::Table table_of(const torch::Tensor& page_table, const torch::Tensor& lens, const torch::Tensor& refs, int page_size) {
  check_int32(page_table, 2, page_table, "page_table");
  check_int32(lens, 1, page_table, "lens");
  check_int32(refs, 1, page_table, "refs");
  TORCH_CHECK_VALUE(lens.size(0) == page_table.size(0), "lens: one entry for each row of page_table");
  return cache::Table{page_table.data_ptr<int>(), lens.data_ptr<int>(), refs.data_ptr<int>(), page_table.stride(0),
                      static_cast<int>(page_table.size(0)), static_cast<int>(page_table.size(1)),
                      static_cast<int>(refs.size(0)), page_size};
}

template <typename S>
S setting(const c10::optional<torch::Tensor>& each, double all, int64_t rows, at::ScalarType type, const torch::Tensor& like,
          const char* what) {
  S s{nullptr, static_cast<decltype(S::all)>(all)};
  if (each) {
    TORCH_CHECK_VALUE(each->device() == like.device() && each->scalar_type() == type && each->dim() == 1 &&
                          each->size(0) == rows && each->is_contiguous(),
                      what, ": a number, or a contiguous ", type, " tensor with one entry for each of the ", rows, " rows");
    s.each = each->data_ptr<decltype(S::all)>();
  }
  return s;
}

}  // namespace

int64_t generation_launches() { return launched; }

void prefix_exp2_eval(const torch::Tensor& x, const torch::Tensor& y) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.scalar_type() == at::kFloat && x.is_contiguous() && x.numel() % 2 == 0 &&
                        x.numel() < (1ll << 31) && y.device() == x.device() && y.sizes() == x.sizes() &&
                        y.scalar_type() == at::kFloat && y.is_contiguous(),
                    "prefix_exp2_eval: contiguous fp32 CUDA tensors of one shape, an even number of entries");
  const c10::cuda::CUDAGuard guard(x.device());
  C10_CUDA_CHECK(prefix::launch_exp2(x.data_ptr<float>(), y.data_ptr<float>(), static_cast<int>(x.numel() / 2),
                                     at::cuda::getCurrentCUDAStream()));
}

void copy_pages(const torch::Tensor& kv, const torch::Tensor& src, const torch::Tensor& dst, const Scales& scales, const torch::Tensor& status) {
  launched = 0;
  const auto p = pool_of(kv, scales);
  check_int32(src, 1, kv, "src");
  check_int32(dst, 1, kv, "dst");
  check_status_word(status);
  TORCH_CHECK_VALUE(src.size(0) == dst.size(0), "src and dst: one destination for each source");
  const c10::cuda::CUDAGuard guard(kv.device());
  C10_CUDA_CHECK(cache::launch_copy(p, src.data_ptr<int>(), dst.data_ptr<int>(), nullptr, nullptr,
                                    static_cast<int>(src.size(0)), errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = src.size(0) > 0;
}

void fork_sequences(const torch::Tensor& kv, const torch::Tensor& page_table, const torch::Tensor& lens, const torch::Tensor& refs,
                    const torch::Tensor& parents, const torch::Tensor& children, const Scales& scales, const torch::Tensor& status) {
  launched = 0;
  const auto p = pool_of(kv, scales);
  const auto t = table_of(page_table, lens, refs, p.page_size);
  check_int32(parents, 1, kv, "parents");
  check_int32(children, 1, kv, "children");
  check_status_word(status);
  TORCH_CHECK_VALUE(page_table.device() == kv.device(), "page_table and kv: on one device");
  TORCH_CHECK_VALUE(refs.size(0) == p.pages, "refs: one count for each page of kv");
  TORCH_CHECK_VALUE(parents.size(0) == children.size(0), "parents and children: one parent for each child");
  const int64_t n = parents.size(0);
  if (n == 0 || t.slots == 0 || t.columns == 0) return;
  TORCH_CHECK_VALUE(n < (1 << 28), "children: too many");
  const c10::cuda::CUDAGuard guard(kv.device());
  auto scratch = at::empty({4 * n + t.slots}, parents.options());
  C10_CUDA_CHECK(cache::launch_fork(p, t, parents.data_ptr<int>(), children.data_ptr<int>(), static_cast<int>(n),
                                    scratch.data_ptr<int>(), errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = 2;
}

void reserve_pages(const torch::Tensor& page_table, const torch::Tensor& lens, const torch::Tensor& refs, const torch::Tensor& slots,
                   const torch::Tensor& counts, int64_t page_size, const torch::Tensor& status) {
  launched = 0;
  TORCH_CHECK_VALUE(page_size >= 1 && page_size < (1 << 30), "page_size: at least 1");
  const auto t = table_of(page_table, lens, refs, static_cast<int>(page_size));
  check_int32(slots, 1, page_table, "slots");
  check_int32(counts, 1, page_table, "counts");
  check_status_word(status);
  TORCH_CHECK_VALUE(slots.size(0) == counts.size(0), "slots and counts: one count for each slot");
  const int64_t n = slots.size(0);
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(page_table.device());
  auto scratch = at::empty({t.pages + n + t.slots}, slots.options());
  C10_CUDA_CHECK(cache::launch_reserve(t, slots.data_ptr<int>(), counts.data_ptr<int>(), static_cast<int>(n),
                                       scratch.data_ptr<int>(), errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = 1;
}

void free_sequences(const torch::Tensor& page_table, const torch::Tensor& lens, const torch::Tensor& refs, const torch::Tensor& slots,
                    const torch::Tensor& status) {
  launched = 0;
  const auto t = table_of(page_table, lens, refs, 1);
  check_int32(slots, 1, page_table, "slots");
  check_status_word(status);
  const int n = static_cast<int>(slots.size(0));
  if (n == 0 || t.columns == 0) return;
  const c10::cuda::CUDAGuard guard(page_table.device());
  C10_CUDA_CHECK(cache::launch_free(t, slots.data_ptr<int>(), n, errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = 1;
}

std::tuple<torch::Tensor, torch::Tensor> compact_pages(const torch::Tensor& kv, const torch::Tensor& page_table, const torch::Tensor& refs,
                                                       const Scales& scales, const torch::Tensor& status) {
  launched = 0;
  const auto p = pool_of(kv, scales);
  check_int32(page_table, 2, kv, "page_table");
  check_int32(refs, 1, kv, "refs");
  check_status_word(status);
  TORCH_CHECK_VALUE(refs.size(0) == p.pages, "refs: one count for each page of kv");
  const c10::cuda::CUDAGuard guard(kv.device());
  auto new_table = at::empty(page_table.sizes(), page_table.options());
  auto new_refs = at::empty(refs.sizes(), refs.options());
  auto scratch = at::empty({3 * static_cast<int64_t>(p.pages) + 1}, refs.options());
  C10_CUDA_CHECK(cache::launch_compact(p, page_table.data_ptr<int>(), page_table.stride(0),
                                       static_cast<int>(page_table.size(0)), static_cast<int>(page_table.size(1)),
                                       refs.data_ptr<int>(), new_table.data_ptr<int>(), new_refs.data_ptr<int>(),
                                       scratch.data_ptr<int>(), errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = page_table.numel() > cache::kSmallTable ? 3 : 2;
  return {new_table, new_refs};
}

void append_kv(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& page_table,
               const torch::Tensor& positions, const c10::optional<torch::Tensor>& slots,
               const Scales& k_scales, const Scales& v_scales, const torch::Tensor& status) {
  launched = 0;
  const auto codes = codes_of(k_pages, v_pages, k_scales, v_scales);
  TORCH_CHECK_VALUE(k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == at::kBFloat16 &&
                        v.scalar_type() == at::kBFloat16 && k.device() == k_pages.device() && v.device() == k.device(),
                    "k and v: bf16 tensors [tokens, kv_heads, head_dim] on the pages' device");
  const int64_t H = k_pages.size(2), D = k_pages.size(3), n = k.size(0);
  TORCH_CHECK_VALUE(k.size(1) == H && k.size(2) == D, "k and v: ", H, " heads of ", D, " as in the pages");
  TORCH_CHECK_VALUE(codes ? D % 16 == 0 && D <= 256 : D % 8 == 0, "head_dim: a multiple of 8 (in 8 bits: of 16, and at most 256)");
  TORCH_CHECK_VALUE(n == 0 || k_pages.numel() == 0 ||
                        (rows_aligned(k) && rows_aligned(v) && rows_aligned(k_pages) && rows_aligned(v_pages)),
                    "k, v and the pages: last axis contiguous, rows 16-byte aligned");
  check_int32(page_table, 2, k_pages, "page_table");
  check_int32(positions, 1, k_pages, "positions");
  check_status_word(status);
  TORCH_CHECK_VALUE(positions.size(0) == n, "positions: one for each token");
  if (slots) {
    check_int32(*slots, 1, k_pages, "slots");
    TORCH_CHECK_VALUE(slots->size(0) == n, "slots: one for each token");
  } else {
    TORCH_CHECK_VALUE(n <= page_table.size(0), "without slots, token i belongs to row i of page_table: too many tokens");
  }
  if (codes)
    TORCH_CHECK_VALUE(k_pages.numel() == 0 || (k_scales->data_ptr() != v_scales->data_ptr() && (k_scales->size(0) <= 1 || k_scales->stride(0) != 0) &&
                                               (H <= 1 || k_scales->stride(1) != 0)),
                      "k_scales and v_scales: memory of their own for each page and head");
  if (n * H * D == 0 || k_pages.size(1) == 0) return;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  TORCH_CHECK_VALUE(n < (1ll << 31), "too many tokens");
  auto fill = [&](auto& a) {
    a.page_ld = k_pages.stride(0);
    a.token_ld = k_pages.stride(1);
    a.head_ld = k_pages.stride(2);
    a.k = bf16(k);
    a.v = bf16(v);
    a.k_ld = k.stride(0);
    a.k_head = k.stride(1);
    a.v_ld = v.stride(0);
    a.v_head = v.stride(1);
    a.table = page_table.data_ptr<int>();
    a.table_ld = page_table.stride(0);
    a.slots = static_cast<int>(page_table.size(0));
    a.columns = static_cast<int>(page_table.size(1));
    a.pages = static_cast<int>(k_pages.size(0));
    a.page_size = static_cast<int>(k_pages.size(1));
    a.positions = positions.data_ptr<int>();
    a.slot_of = slots ? slots->data_ptr<int>() : nullptr;
    a.n = static_cast<int>(n);
    a.heads = static_cast<int>(H);
  };
  if (codes) {
    cache::Append8 a{};
    a.e4m3 = codes == prefix::kE4m3;
    a.k_pool = bytes(k_pages);
    a.v_pool = bytes(v_pages);
    a.k_scales = k_scales->data_ptr<float>();
    a.v_scales = v_scales->data_ptr<float>();
    a.scale_ld = k_scales->stride(0);
    a.scale_head = k_scales->stride(1);
    a.dim = static_cast<int>(D);
    fill(a);
    C10_CUDA_CHECK(cache::launch_append8(a, errors_of(status), at::cuda::getCurrentCUDAStream()));
    launched = 1;
    return;
  }
  cache::Append a{};
  a.k_pool = bf16(k_pages);
  a.v_pool = bf16(v_pages);
  fill(a);
  a.chunks = static_cast<int>(D / 8);
  C10_CUDA_CHECK(cache::launch_append(a, errors_of(status), at::cuda::getCurrentCUDAStream()));
  launched = 1;
}

std::tuple<torch::Tensor, c10::optional<torch::Tensor>> sample(
    const torch::Tensor& logits, const torch::Tensor& noise, const c10::optional<torch::Tensor>& temperature, double temperature_all,
    const c10::optional<torch::Tensor>& top_k, int64_t top_k_all, const c10::optional<torch::Tensor>& top_p, double top_p_all,
    const c10::optional<torch::Tensor>& min_p, double min_p_all, bool return_logprob, const torch::Tensor& status) {
  launched = 0;
  using sampling::Setting;
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 &&
                        (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
                    "logits: a bf16 or fp32 tensor [rows, vocabulary]");
  const int64_t R = logits.size(0), V = logits.size(1);
  TORCH_CHECK_VALUE(V >= 1 && V <= (1 << sampling::kIndexBits), "vocabulary: 1 to 1048576 tokens, got ", V);
  TORCH_CHECK_VALUE(logits.stride(1) == 1 || V == 1, "logits: last axis contiguous");
  TORCH_CHECK_VALUE(noise.device() == logits.device() && noise.scalar_type() == at::kFloat && noise.sizes() == logits.sizes() &&
                        (noise.stride(1) == 1 || V == 1),
                    "noise: an fp32 tensor of the logits' shape, last axis contiguous");
  TORCH_CHECK_VALUE(R < (1ll << 31), "too many rows");
  check_status_word(status);
  sampling::Sample a{};
  a.status = waits_of(status);
  a.temperature = setting<Setting>(temperature, temperature_all, R, at::kFloat, logits, "temperature");
  a.top_k = setting<sampling::WholeSetting>(top_k, static_cast<double>(std::clamp<int64_t>(top_k_all, 0, V)), R, at::kInt,
                                            logits, "top_k");
  a.top_p = setting<Setting>(top_p, top_p_all, R, at::kFloat, logits, "top_p");
  a.min_p = setting<Setting>(min_p, min_p_all, R, at::kFloat, logits, "min_p");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto token = at::empty({R}, logits.options().dtype(at::kLong));
  c10::optional<torch::Tensor> logprob;
  if (return_logprob) logprob = at::empty({R}, logits.options().dtype(at::kFloat));
  if (R == 0) return {token, logprob};
  a.logits = logits.data_ptr();
  a.bf16 = logits.scalar_type() == at::kBFloat16;
  a.ld = logits.stride(0);
  a.noise = noise.data_ptr<float>();
  a.noise_ld = noise.stride(0);
  a.rows = static_cast<int>(R);
  a.vocab = static_cast<int>(V);
  a.token = reinterpret_cast<long long*>(token.data_ptr<int64_t>());
  a.logprob = logprob ? logprob->data_ptr<float>() : nullptr;
  C10_CUDA_CHECK(sampling::launch_sample(a, at::cuda::getCurrentCUDAStream()));
  launched = 1;
  return {token, logprob};
}

namespace {

// A list of tokens for each row, or one for all of them.
logits::Ids ids_of(const c10::optional<torch::Tensor>& t, int64_t rows, const torch::Tensor& like, bool shared, const char* what) {
  logits::Ids ids{};
  if (!t) return ids;
  TORCH_CHECK_VALUE(t->device() == like.device() && (t->scalar_type() == at::kLong || t->scalar_type() == at::kInt) &&
                        ((t->dim() == 2 && t->size(0) == rows) || (shared && t->dim() == 1)) &&
                        (t->numel() == 0 || t->size(-1) == 1 || t->stride(-1) == 1),
                    what, ": int64 or int32 tokens [", rows, " rows, n]", shared ? " or [n]" : "", " on the logits' device, last axis contiguous");
  ids.ids = t->data_ptr();
  ids.wide = t->scalar_type() == at::kLong;
  ids.ld = t->dim() == 2 ? t->stride(0) : 0;
  ids.n = t->size(-1);
  return ids;
}

}  // namespace

torch::Tensor adjust_logits(const torch::Tensor& in, const c10::optional<torch::Tensor>& given, const c10::optional<torch::Tensor>& prompt,
                   const c10::optional<torch::Tensor>& history, const c10::optional<torch::Tensor>& history_lens,
                   const c10::optional<torch::Tensor>& repetition, double repetition_all, const c10::optional<torch::Tensor>& presence,
                   double presence_all, const c10::optional<torch::Tensor>& frequency, double frequency_all,
                   const c10::optional<torch::Tensor>& bias_tokens, const c10::optional<torch::Tensor>& bias,
                   const c10::optional<torch::Tensor>& allowed, const c10::optional<torch::Tensor>& mask_of, const torch::Tensor& status) {
  launched = 0;
  using sampling::Setting;
  TORCH_CHECK_VALUE(in.is_cuda() && in.dim() == 2 && (in.scalar_type() == at::kBFloat16 || in.scalar_type() == at::kFloat),
                    "logits: a bf16 or fp32 tensor [rows, vocabulary]");
  const int64_t R = in.size(0), V = in.size(1);
  TORCH_CHECK_VALUE(V >= 1 && V <= (1 << sampling::kIndexBits), "vocabulary: 1 to 1048576 tokens, got ", V);
  TORCH_CHECK_VALUE(in.stride(1) == 1 || V == 1, "logits: last axis contiguous");
  const torch::Tensor out = given ? *given : at::empty(in.sizes(), in.options());
  TORCH_CHECK_VALUE(out.device() == in.device() && out.scalar_type() == in.scalar_type() && out.sizes() == in.sizes() &&
                        (out.stride(1) == 1 || V == 1) && (R <= 1 || out.stride(0) >= V),
                    "out: a tensor like logits, last axis contiguous, rows apart");
  check_status_word(status);
  logits::Adjust a{};
  a.prompt = ids_of(prompt, R, in, true, "prompt");
  a.history = ids_of(history, R, in, false, "history");
  a.bias_tokens = ids_of(bias_tokens, R, in, true, "bias_tokens");
  TORCH_CHECK_VALUE(a.history.n < (1 << logits::kCountBits) && a.prompt.n < (1ll << 31), "history: at most ", (1 << logits::kCountBits) - 1, " tokens a row");
  if (history_lens) {
    check_int32(*history_lens, 1, in, "history_lens");
    TORCH_CHECK_VALUE(history && history_lens->size(0) == R, "history_lens: one length for each row of history");
    TORCH_CHECK_VALUE(history_lens->is_contiguous(), "history_lens: contiguous");
    a.history_lens = history_lens->data_ptr<int>();
  }
  TORCH_CHECK_VALUE(bias_tokens.has_value() == bias.has_value(), "bias_tokens and bias: one needs the other");
  if (bias) {
    TORCH_CHECK_VALUE(bias->device() == in.device() && bias->scalar_type() == at::kFloat && bias->sizes() == bias_tokens->sizes() &&
                          bias->is_contiguous() && bias_tokens->is_contiguous(),
                      "bias_tokens and bias: contiguous, fp32 biases of the tokens' shape");
    TORCH_CHECK_VALUE(a.bias_tokens.n <= logits::kMostBiases, "bias_tokens: at most ", logits::kMostBiases, " a row");
    a.bias = bias->data_ptr<float>();
  }
  a.repetition = setting<Setting>(repetition, repetition_all, R, at::kFloat, in, "repetition");
  a.presence = setting<Setting>(presence, presence_all, R, at::kFloat, in, "presence");
  a.frequency = setting<Setting>(frequency, frequency_all, R, at::kFloat, in, "frequency");
  if (allowed) {
    check_int32(*allowed, 2, in, "allowed");
    TORCH_CHECK_VALUE(allowed->size(1) == (V + 31) / 32, "allowed: ", (V + 31) / 32, " words of 32 tokens a mask");
    a.allowed = reinterpret_cast<const uint32_t*>(allowed->data_ptr<int>());
    a.mask_ld = allowed->stride(0);
    a.masks = static_cast<int>(allowed->size(0));
    if (mask_of) {
      check_int32(*mask_of, 1, in, "mask_of");
      TORCH_CHECK_VALUE(mask_of->size(0) == R && mask_of->is_contiguous(), "mask_of: contiguous, one mask for each row");
      a.mask_of = mask_of->data_ptr<int>();
    } else {
      TORCH_CHECK_VALUE(a.masks == 1 || a.masks == R, "allowed: without mask_of one mask, or one for each row");
    }
  } else {
    TORCH_CHECK_VALUE(!mask_of, "mask_of: needs allowed");
  }
  if (R == 0) return out;
  TORCH_CHECK_VALUE(R * ((V + 2047) / 2048 + 1) < (1ll << 31), "too many rows");
  const c10::cuda::CUDAGuard guard(in.device());
  a.in = in.data_ptr();
  a.out = out.data_ptr();
  a.bf16 = in.scalar_type() == at::kBFloat16;
  a.in_ld = in.stride(0);
  a.out_ld = out.stride(0);
  a.in_place = a.in == a.out && (a.in_ld == a.out_ld || R == 1);
  auto end_of = [&](const torch::Tensor& t) { return static_cast<const char*>(t.data_ptr()) + ((R - 1) * t.stride(0) + V) * t.element_size(); };
  TORCH_CHECK_VALUE(a.in_place || end_of(in) <= static_cast<const char*>(out.data_ptr()) || end_of(out) <= static_cast<const char*>(in.data_ptr()),
                    "out: logits itself, or memory that does not overlap it");
  a.rows = static_cast<int>(R);
  a.vocab = static_cast<int>(V);
  a.status = errors_of(status);
  C10_CUDA_CHECK(logits::launch_adjust(a, at::cuda::getCurrentCUDAStream()));
  launched = 1;
  return out;
}

std::tuple<torch::Tensor, c10::optional<torch::Tensor>> shared_prefix_attention(
    const torch::Tensor& q, const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& prefix_pages, int64_t prefix_len,
    const torch::Tensor& page_table, const torch::Tensor& seq_lens, const c10::optional<torch::Tensor>& q_offsets, int64_t max_q_len,
    int64_t max_seq_len, double scale, bool return_lse, const Scales& k_scales, const Scales& v_scales, const torch::Tensor& status) {
  launched = 0;
  TORCH_CHECK_VALUE(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3,
                    "q: a bf16 CUDA tensor [tokens, heads, head_dim]");
  const auto codes = codes_of(k_pages, v_pages, k_scales, v_scales);
  TORCH_CHECK_VALUE(k_pages.device() == q.device(), "k_pages and v_pages: on q's device");
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2);
  const int64_t pages = k_pages.size(0), page = k_pages.size(1), Hk = k_pages.size(2);
  TORCH_CHECK_VALUE(D == 32 || D == 64 || D == 128, "head_dim: 32, 64 or 128, got ", D);
  TORCH_CHECK_VALUE(k_pages.size(3) == D, "k_pages: head_dim ", D, " as in q, got ", k_pages.size(3));
  TORCH_CHECK_VALUE(Hk > 0 && H > 0 && H % Hk == 0, "heads: a multiple of the pages' ", Hk, " kv heads, got ", H);
  TORCH_CHECK_VALUE(page >= 8 && page <= 256 && (page & (page - 1)) == 0, "page_size: a power of two from 8 to 256, got ", page);
  TORCH_CHECK_VALUE(N == 0 || rows_aligned(q), "q: last axis contiguous, rows 16-byte aligned");
  TORCH_CHECK_VALUE(pages == 0 || (rows_aligned(k_pages) && rows_aligned(v_pages)),
                    "pages: last axis contiguous, rows 16-byte aligned");
  for (int64_t i = 0; i < 3; ++i)
    TORCH_CHECK_VALUE(k_pages.size(i) <= 1 || (k_pages.stride(i) > 0 && k_pages.stride(i) < (1ll << 39)),
                      "pages: an axis with a stride that a tensor map cannot hold (expanded?)");
  check_int32(prefix_pages, 1, q, "prefix_pages");
  check_int32(page_table, 2, q, "page_table");
  check_int32(seq_lens, 1, q, "seq_lens");
  check_status_word(status);
  const int64_t B = page_table.size(0);
  TORCH_CHECK_VALUE(seq_lens.size(0) == B, "seq_lens: one length for each row of page_table");
  TORCH_CHECK_VALUE(prefix_len >= 0 && prefix_len <= prefix_pages.size(0) * page, "prefix_len: 0 to the ",
                    prefix_pages.size(0) * page, " tokens of prefix_pages, got ", prefix_len);
  const int64_t room = page_table.size(1) * page;
  if (max_seq_len < 0) max_seq_len = room;
  TORCH_CHECK_VALUE(max_seq_len <= room, "max_seq_len: at most the ", room, " tokens of a row of page_table, got ", max_seq_len);
  if (q_offsets) {
    check_int32(*q_offsets, 1, q, "q_offsets");
    TORCH_CHECK_VALUE(q_offsets->size(0) == B + 1, "q_offsets: one more entry than page_table has rows");
    TORCH_CHECK_VALUE(max_q_len >= 0, "max_q_len: needed with q_offsets");
    TORCH_CHECK_VALUE(N == 0 || B > 0, "q_offsets: no sequence for the ", N, " tokens");
    TORCH_CHECK_VALUE(N == 0 || max_q_len > 0, "max_q_len: at least 1 for ", N, " tokens");
  } else {
    TORCH_CHECK_VALUE(N == B, "without q_offsets there is one token for each of the ", B, " sequences, got ", N);
    max_q_len = 1;
  }
  TORCH_CHECK_VALUE(N * H < (1ll << 31) && prefix_len < (1ll << 30) && room < (1ll << 30), "too many rows or keys");

  const c10::cuda::CUDAGuard guard(q.device());
  auto o = at::empty({N, H, D}, q.options());
  c10::optional<torch::Tensor> lse;
  if (return_lse) lse = at::empty({N, H}, q.options().dtype(at::kFloat));
  if (N == 0) return {o, lse};

  prefix::Args a{};
  a.q = bf16(q);
  a.q_ld = q.stride(0);
  a.q_head = q.stride(1);
  // (a map needs an address, also where nothing will be read)
  const torch::Tensor &k_of = pages > 0 ? k_pages : q, &v_of = pages > 0 ? v_pages : q;
  a.codes = codes;
  if (codes) {
    a.k8 = bytes(k_of);
    a.v8 = bytes(v_of);
    // (an address also where there are no pages and nothing will be read)
    a.k_scales = pages > 0 ? k_scales->data_ptr<float>() : reinterpret_cast<const float*>(q.data_ptr());
    a.v_scales = pages > 0 ? v_scales->data_ptr<float>() : a.k_scales;
    a.scale_ld = k_scales->stride(0);
    a.scale_head = k_scales->stride(1);
  } else {
    a.k = bf16(k_of);
    a.v = bf16(v_of);
  }
  a.page_ld = k_pages.stride(0);
  a.token_ld = k_pages.stride(1);
  a.head_ld = k_pages.stride(2);
  a.pages = static_cast<int>(pages);
  a.no_page = std::max(1, a.pages);  // (a map has at least one page)
  a.page_shift = __builtin_ctzll(static_cast<uint64_t>(page));
  a.prefix_pages = prefix_pages.data_ptr<int>();
  a.prefix_len = static_cast<int>(prefix_len);
  a.page_table = page_table.data_ptr<int>();
  a.table_ld = page_table.stride(0);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.q_offsets = q_offsets ? q_offsets->data_ptr<int>() : nullptr;
  a.n = static_cast<int>(N);
  a.batch = static_cast<int>(B);
  a.kv_heads = static_cast<int>(Hk);
  a.heads = static_cast<int>(H);
  a.group = static_cast<int>(H / Hk);
  a.max_q = static_cast<int>(std::min(max_q_len, N));
  a.max_len = static_cast<int>(max_seq_len);
  a.scale_log2 = static_cast<float>(scale * kLog2e);
  a.status = waits_of(status);
  a.errors = errors_of(status);
  a.o = bf16(o);
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  const int64_t pieces = prefix::plan(a, static_cast<int>(D)), rows = N * H;
  TORCH_CHECK_VALUE(B * a.own_tiles * a.own_splits * Hk < (1ll << 30), "too many sequences times max_q_len");
  TORCH_CHECK_VALUE(static_cast<int64_t>(a.row_tiles) * a.prefix_splits * Hk < (1ll << 30), "too many rows");
  torch::Tensor part;
  if (pieces > 0) {
    part = at::empty({pieces * rows * (D + 2) + 1}, q.options().dtype(at::kFloat));
    a.part_o = part.data_ptr<float>();
    a.part_ml = reinterpret_cast<float2*>(a.part_o + pieces * rows * D);
    if (q_offsets && a.own_splits > 0) a.sound = reinterpret_cast<int*>(a.part_ml + pieces * rows);
  }
  C10_CUDA_CHECK(prefix::launch_attention(a, static_cast<int>(D), at::cuda::getCurrentCUDAStream()));
  launched = prefix::kernels(a);
  return {o, lse};
}

}  // namespace mnb
