// Host path of the serving operators for PyTorch: argument checks, outputs and
// workspaces, and the calls of the C ABI, without the interpreter.  A decode step
// makes a few of these calls per layer and its kernels take microseconds each.
//
// What is read on the device (lengths, page ids, slots, starts, counts) is checked
// there; what can be seen on the host is checked here: ValueError for shapes and
// numbers, TypeError for dtypes, RuntimeError for tensors on the wrong device.
//
// Tensors that are not of the ordinary kind, and calls that a tracer, mode or transform
// looks at, are left to the library ops, which those can see: None comes back.
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <optional>

#include "../../../include/nanochat_decoding_amd.h"
#include "../../../include/nanochat_serving_amd.h"
#include "ltv_torch.hpp"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;
using OptInt = std::optional<int64_t>;

void check_rc(int rc, const char* what) {
  static const char* names[] = {"LTV_OK", "LTV_ERR_INVALID_ARG", "LTV_ERR_UNSUPPORTED",
                                "LTV_ERR_HIP", "LTV_ERR_WORKSPACE"};
  if (rc == 0) return;
  const std::string name = rc > 0 && rc < 5 ? names[rc] : std::to_string(rc);
  TORCH_CHECK(false, what, " failed (", name, "): ", ltv_last_error());
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A call's workspace: torch's caching allocator without a tensor around it (a microsecond
// less), on the current stream of the current device; given back when the call has been
// made, which is in order with later users of the stream.
struct Workspace {
  c10::DataPtr mem;
  size_t bytes;
  explicit Workspace(size_t n) : bytes(n) {
    if (n > 0) mem = c10::hip::HIPCachingAllocator::get()->allocate(n);
  }
  void* ptr() const { return bytes > 0 ? mem.get() : nullptr; }
};

bool ordinary(const Tensor& t) {
  return !at::isTensorSubclassLike(t) && !t.is_neg() && !t._is_zerotensor();
}
bool ordinary(const OptTensor& t) { return !t.has_value() || ordinary(*t); }

// (a mode is seen by each tensor's check)
template <typename... Ts>
bool ordinary_call(const Ts&... ts) {
  return !torch::jit::tracer::isTracing() && (ordinary(ts) && ...);
}

// (asked before a call goes to a library op: there a transform's tangents are just dropped)
void no_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
                t._fw_grad(/*level=*/0).defined()),
              name, " has a tangent, but there is no forward-mode derivative");
}

void on_device(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), "LTV HIP kernels need GPU tensors, got ", name, " on ", t.device());
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", the others on ",
              like.device());
}

int dtype_of(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16,
                   "LTV kernels support float32 and bfloat16 tensors, got ", name, " of ",
                   t.scalar_type());
  return t.scalar_type() == at::kFloat ? LTV_DTYPE_F32 : LTV_DTYPE_BF16;
}

int to_int(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v <= std::numeric_limits<int>::max(), name, " is out of range: ",
                    v);
  return (int)v;
}

// An int32 vector on like's device, contiguous (int64 ones are converted; what 32 bits do
// not hold becomes their end, which is out of every range, and not an id that is in one).
Tensor int_vector(const Tensor& t, const char* name, const Tensor& like) {
  on_device(t, name, like);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name,
                   " must be int32 or int64, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1, name, " must be a vector, got ", t.sizes());
  if (t.scalar_type() == at::kInt) return t.contiguous();
  using lim = std::numeric_limits<int32_t>;
  return t.clamp(lim::min(), lim::max()).to(at::kInt).contiguous();
}

// The cache's own tables are read, or written, where they are.
void int_table(const Tensor& t, const char* name, int dim, const Tensor& like) {
  on_device(t, name, like);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dim && (t.numel() == 0 || t.stride(dim - 1) == 1), name,
                    " must have ", dim, " dimensions, the last one contiguous");
}

// Whether pages are 4-bit ones, whose elements are bytes.
bool is_fp4(const Tensor& pages) { return pages.scalar_type() == at::kByte; }

// 4-bit pages of one layer, (P, NKVH, page, D / 2 + D / 32).
void check_fp4_pages(const Tensor& k, const Tensor& v, const Tensor& like) {
  on_device(k, "k_pages", like);
  on_device(v, "v_pages", like);
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(),
                    "k_pages and v_pages must be (pages, kv heads, page size, bytes of a token) and "
                    "alike, got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(is_fp4(k) && is_fp4(v), "k_pages are ", k.scalar_type(), ", v_pages ",
                   v.scalar_type());
  const int64_t row = k.size(3);
  TORCH_CHECK_VALUE(row % 17 == 0 && row >= 17 && row <= 68,
                    "a token's head takes 17 bytes for each 32 of a head_dim of 32 to 128 in 4 bits, "
                    "got ", row);
  TORCH_CHECK_VALUE(k.size(2) > 0 && k.size(2) % 16 == 0,
                    "a 4-bit page must hold a multiple of 16 tokens, got ", k.size(2));
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK_VALUE(
        t->numel() == 0 ||
            (t->stride(3) == 1 && t->stride(2) == row && (t->size(0) == 1 || t->stride(0) % 16 == 0) &&
             (t->size(1) == 1 || t->stride(1) % 16 == 0) &&
             reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0),
        "4-bit pages must be dense blocks of a page and head, 16-byte aligned");
}

// Pages of one layer, (P, NKVH, page, D).
void check_pages(const Tensor& k, const Tensor& v, const Tensor& like) {
  on_device(k, "k_pages", like);
  on_device(v, "v_pages", like);
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(),
                    "k_pages and v_pages must be (pages, kv heads, page size, head_dim) and alike, "
                    "got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(k.scalar_type() == like.scalar_type() && v.scalar_type() == k.scalar_type(),
                   "the pages must have the tokens' dtype ", like.scalar_type(), ", got ",
                   k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK_VALUE(k.size(2) > 0, "a page must hold tokens");
  const int64_t align = 16 / k.element_size();
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK_VALUE(
        t->numel() == 0 ||
            (t->stride(3) == 1 && t->stride(0) % align == 0 && t->stride(1) % align == 0 &&
             t->stride(2) % align == 0 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0),
        "the pages' rows must be contiguous and 16-byte aligned");
}

struct Batch {
  ltv_paged_batch b{};
  Tensor table, slots, starts;  // (kept until the call has been made)
};

// A table whose rows lie one after the other, not in each other (an expanded row).
bool rows_apart(const Tensor& t) { return t.size(0) <= 1 || t.stride(0) >= t.size(1); }

// tok: the token tensor, (B, T, heads, D) or, with starts, (N, heads, D)
Batch make_batch(const Tensor& tok, const char* name, const Tensor& k_pages, const Tensor& table,
                 const Tensor& lens, const OptTensor& slots, const OptTensor& starts,
                 const OptInt& max_new) {
  Batch r;
  int_table(table, "page_table", 2, tok);
  int_table(lens, "seq_lens", 1, tok);
  TORCH_CHECK_VALUE(lens.size(0) == table.size(0), "page_table has ", table.size(0),
                    " rows, seq_lens ", lens.size(0));
  r.table = rows_apart(table) ? table : table.contiguous();
  r.b.page_table = table.numel() ? r.table.data_ptr<int32_t>() : nullptr;
  r.b.seq_lens = lens.numel() ? lens.data_ptr<int32_t>() : nullptr;
  r.b.table_stride = std::max(r.table.stride(0), table.size(1));
  r.b.num_slots = to_int(table.size(0), "the number of slots");
  r.b.table_width = to_int(table.size(1), "the page table's width");
  r.b.num_pages = to_int(k_pages.size(0), "the number of pages");
  r.b.page_size = to_int(k_pages.size(2), "the page size");
  int64_t B;
  if (starts.has_value()) {
    TORCH_CHECK_VALUE(tok.dim() == 3, "with starts, ", name, " must be (tokens, heads, head_dim), "
                      "got ", tok.sizes());
    r.starts = int_vector(*starts, "starts", tok);
    TORCH_CHECK_VALUE(r.starts.numel() >= 1, "starts must have one entry more than sequences");
    r.b.starts = r.starts.data_ptr<int32_t>();
    B = r.starts.numel() - 1;
    r.b.total = tok.size(0);
    TORCH_CHECK_VALUE(!max_new.has_value() || *max_new >= 0, "max_new is negative");
    r.b.T = to_int(std::min(max_new.value_or(tok.size(0)), tok.size(0)), "max_new");
  } else {
    TORCH_CHECK_VALUE(tok.dim() == 4, name, " must be (batch, tokens, heads, head_dim), got ",
                      tok.sizes());
    TORCH_CHECK_VALUE(!max_new.has_value() || *max_new == tok.size(1), "max_new is ",
                      max_new.value_or(0), ", but each sequence has ", tok.size(1), " new tokens");
    B = tok.size(0);
    r.b.T = to_int(tok.size(1), "the number of new tokens");
    r.b.total = B * tok.size(1);
  }
  r.b.B = to_int(B, "the number of sequences");
  if (slots.has_value()) {
    r.slots = int_vector(*slots, "slots", tok);
    TORCH_CHECK_VALUE(r.slots.numel() == B, r.slots.numel(), " slots for ", B, " sequences");
    r.b.slots = r.slots.data_ptr<int32_t>();
  } else {
    TORCH_CHECK_VALUE(B <= table.size(0), B, " sequences, but page_table has ", table.size(0),
                      " rows");
  }
  return r;
}

struct Strides3 {
  int64_t s[3];
  // (sequence, token, head) strides of a token tensor
  static Strides3 tokens(const Tensor& t) {
    return t.dim() == 4 ? Strides3{{t.stride(0), t.stride(1), t.stride(2)}}
                        : Strides3{{0, t.stride(0), t.stride(1)}};
  }
  static Strides3 pages(const Tensor& t) { return {{t.stride(0), t.stride(1), t.stride(2)}}; }
  // (an axis of one element has no stride to speak of)
  static Strides3 fp4_pages(const Tensor& t) {
    return {{t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1), t.size(3)}};
  }
};

Tensor rows_contiguous(const Tensor& t) {
  return t.numel() == 0 || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

int64_t head_dim_of(const Tensor& pages) {
  return is_fp4(pages) ? pages.size(3) / 17 * 32 : pages.size(3);
}

void check_any_pages(const Tensor& k, const Tensor& v, const Tensor& like) {
  if (is_fp4(k)) check_fp4_pages(k, v, like);
  else check_pages(k, v, like);
}

Strides3 any_strides(const Tensor& pages) {
  return is_fp4(pages) ? Strides3::fp4_pages(pages) : Strides3::pages(pages);
}

void no_grad_needed(const Tensor& t, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires grad, but the paged cache is for inference: call under torch.no_grad()");
}

// ---------------------------------------------------------------------------
// the cache
// ---------------------------------------------------------------------------
bool append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_pages, const Tensor& v_pages,
            const Tensor& table, const Tensor& lens, const OptTensor& slots,
            const OptTensor& starts, const OptInt& max_new) {
  no_tangent(k_in, "k");
  no_tangent(v_in, "v");
  if (!ordinary_call(k_in, v_in, k_pages, v_pages, table, lens, slots, starts)) return false;
  const int dt = dtype_of(k_in, "k");
  TORCH_CHECK(k_in.is_cuda(), "LTV HIP kernels need GPU tensors, got k on ", k_in.device());
  on_device(v_in, "v", k_in);
  no_grad_needed(k_in, "k");
  no_grad_needed(v_in, "v");
  check_any_pages(k_pages, v_pages, k_in);
  const Batch b = make_batch(k_in, "k", k_pages, table, lens, slots, starts, max_new);
  TORCH_CHECK_VALUE(v_in.sizes() == k_in.sizes(), "k is ", k_in.sizes(), ", v ", v_in.sizes());
  TORCH_CHECK_TYPE(v_in.scalar_type() == k_in.scalar_type(), "k is ", k_in.scalar_type(), ", v ",
                   v_in.scalar_type());
  const int64_t heads = k_pages.size(1), D = head_dim_of(k_pages);
  TORCH_CHECK_VALUE(k_in.size(-2) == heads && k_in.size(-1) == D, "the pages hold ", heads,
                    " heads of ", D, ", k is ", k_in.sizes());
  const Tensor k = rows_contiguous(k_in), v = rows_contiguous(v_in);
  c10::OptionalDeviceGuard guard(k.device());
  const Strides3 ks = Strides3::tokens(k), vs = Strides3::tokens(v),
                 kp = any_strides(k_pages), vp = any_strides(v_pages);
  if (is_fp4(k_pages)) {
    check_rc(ltv_paged_cache_append_fp4(dt, k.data_ptr(), ks.s, v.data_ptr(), vs.s,
                                        k_pages.data_ptr(), kp.s, v_pages.data_ptr(), vp.s, &b.b,
                                        (int)heads, (int)D, stream_of(k)),
             "ltv_paged_cache_append_fp4");
    return true;
  }
  check_rc(ltv_paged_cache_append(dt, k.data_ptr(), ks.s, v.data_ptr(), vs.s, k_pages.data_ptr(),
                                  kp.s, v_pages.data_ptr(), vp.s, &b.b, (int)heads, (int)D,
                                  stream_of(k)),
           "ltv_paged_cache_append");
  return true;
}

// (the rotated queries)
OptTensor rotary_append(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                        const Tensor& cos_in, const Tensor& sin_in, const Tensor& k_pages,
                        const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                        const OptTensor& slots, const OptTensor& starts, const OptInt& max_new,
                        std::optional<double> norm_eps) {
  no_tangent(q_in, "q");
  no_tangent(k_in, "k");
  no_tangent(v_in, "v");
  no_tangent(cos_in, "cos");
  no_tangent(sin_in, "sin");
  if (!ordinary_call(q_in, k_in, v_in, cos_in, sin_in, k_pages, v_pages, table, lens, slots, starts))
    return {};
  const int dt = dtype_of(q_in, "q");
  TORCH_CHECK(q_in.is_cuda(), "LTV HIP kernels need GPU tensors, got q on ", q_in.device());
  const std::pair<const Tensor*, const char*> others[] = {
      {&k_in, "k"}, {&v_in, "v"}, {&cos_in, "cos"}, {&sin_in, "sin"}};
  for (auto [t, name] : others) on_device(*t, name, q_in);
  no_grad_needed(q_in, "q");
  for (auto [t, name] : others) no_grad_needed(*t, name);
  check_any_pages(k_pages, v_pages, q_in);
  const Batch b = make_batch(q_in, "q", k_pages, table, lens, slots, starts, max_new);
  TORCH_CHECK_VALUE(v_in.sizes() == k_in.sizes(), "k is ", k_in.sizes(), ", v ", v_in.sizes());
  TORCH_CHECK_TYPE(k_in.scalar_type() == q_in.scalar_type() &&
                       v_in.scalar_type() == q_in.scalar_type(),
                   "q is ", q_in.scalar_type(), ", k ", k_in.scalar_type(), ", v ",
                   v_in.scalar_type());
  const int64_t NH = q_in.size(-2), NKVH = k_pages.size(1), D = head_dim_of(k_pages);
  TORCH_CHECK_VALUE(k_in.dim() == q_in.dim() &&
                        k_in.sizes().slice(0, k_in.dim() - 2) ==
                            q_in.sizes().slice(0, q_in.dim() - 2),
                    "q and k must have the same tokens, got ", q_in.sizes(), " and ", k_in.sizes());
  TORCH_CHECK_VALUE(k_in.size(-2) == NKVH && k_in.size(-1) == D && q_in.size(-1) == D,
                    "the pages hold ", NKVH, " heads of ", D, ", k is ", k_in.sizes(), ", q ",
                    q_in.sizes());
  TORCH_CHECK_VALUE(D > 0 && D <= 128 && D % 8 == 0,
                    "head_dim must be a multiple of 8, at most 128, got ", D);
  const int tdt = dtype_of(cos_in, "cos");
  TORCH_CHECK_TYPE(sin_in.scalar_type() == cos_in.scalar_type(), "cos is ", cos_in.scalar_type(),
                   ", sin ", sin_in.scalar_type());
  TORCH_CHECK_VALUE(cos_in.dim() == 2 && cos_in.size(1) == D / 2 && sin_in.sizes() == cos_in.sizes(),
                    "cos and sin must be (positions, ", D / 2, "), got ", cos_in.sizes(), " and ",
                    sin_in.sizes());
  TORCH_CHECK_VALUE(cos_in.size(0) >= (int64_t)b.b.table_width * b.b.page_size, "cos and sin have ",
                    cos_in.size(0), " positions, but the page table has room for ",
                    (int64_t)b.b.table_width * b.b.page_size);
  TORCH_CHECK_VALUE(!norm_eps.has_value() ||
                        (*norm_eps >= 0 && std::isfinite(*norm_eps)),
                    "norm_eps must be finite and not negative, got ",
                    norm_eps.value_or(0));
  const Tensor q = rows_contiguous(q_in), k = rows_contiguous(k_in), v = rows_contiguous(v_in),
               cos = rows_contiguous(cos_in), sin = rows_contiguous(sin_in);
  c10::OptionalDeviceGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
  const Strides3 qs = Strides3::tokens(q), ks = Strides3::tokens(k), vs = Strides3::tokens(v),
                 os = Strides3::tokens(out), kp = any_strides(k_pages), vp = any_strides(v_pages);
  check_rc(ltv_paged_rotary_append(
               dt, q.data_ptr(), qs.s, k.data_ptr(), ks.s, v.data_ptr(), vs.s, cos.data_ptr(),
               cos.stride(0), sin.data_ptr(), sin.stride(0), tdt, cos.size(0),
               norm_eps.value_or(-1.0), out.data_ptr(), os.s,
               k_pages.data_ptr(), kp.s, v_pages.data_ptr(), vp.s,
               is_fp4(k_pages) ? LTV_PAGES_FP4 : LTV_PAGES_VALUES, &b.b, (int)NH, (int)NKVH, (int)D,
               stream_of(q)),
           "ltv_paged_rotary_append");
  return out;
}

// What the pages hold of the new tokens, in dtype.
std::optional<std::tuple<Tensor, Tensor>> read_pages(
    const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
    int64_t tokens, const OptTensor& slots, const OptTensor& starts, const OptInt& max_new,
    at::ScalarType dtype) {
  no_tangent(k_pages, "k_pages");
  no_tangent(v_pages, "v_pages");
  if (!ordinary_call(k_pages, v_pages, table, lens, slots, starts)) return {};
  TORCH_CHECK(k_pages.is_cuda(), "LTV HIP kernels need GPU tensors, got k_pages on ",
              k_pages.device());
  if (!is_fp4(k_pages)) dtype_of(k_pages, "k_pages");
  no_grad_needed(k_pages, "k_pages");
  no_grad_needed(v_pages, "v_pages");
  check_any_pages(k_pages, v_pages, k_pages);
  TORCH_CHECK_TYPE(dtype == at::kFloat || dtype == at::kBFloat16,
                   "LTV kernels support float32 and bfloat16 tensors, got dtype ", dtype);
  TORCH_CHECK_TYPE(is_fp4(k_pages) || dtype == k_pages.scalar_type(), "the pages are ",
                   k_pages.scalar_type(), ", and are read as that, got dtype ", dtype);
  TORCH_CHECK_VALUE(tokens >= 0, "a negative number of tokens: ", tokens);
  const int64_t NKVH = k_pages.size(1), D = head_dim_of(k_pages);
  TORCH_CHECK_VALUE(D > 0 && D <= 128 && D % 8 == 0,
                    "head_dim must be a multiple of 8, at most 128, got ", D);
  c10::OptionalDeviceGuard guard(k_pages.device());
  const auto options = k_pages.options().dtype(dtype).requires_grad(false);
  auto shape = [&]() -> std::vector<int64_t> {
    if (starts.has_value()) return {tokens, NKVH, D};
    return {slots.has_value() ? slots->numel() : table.dim() > 0 ? table.size(0) : 0, tokens, NKVH, D};
  }();
  Tensor k = at::empty(shape, options), v = at::empty(shape, options);
  const Batch b = make_batch(k, "the result", k_pages, table, lens, slots, starts, max_new);
  if (k.numel() == 0) return std::make_tuple(k, v);
  const Strides3 kp = any_strides(k_pages), vp = any_strides(v_pages);
  check_rc(ltv_paged_cache_read(dtype == at::kFloat ? LTV_DTYPE_F32 : LTV_DTYPE_BF16,
                                is_fp4(k_pages) ? LTV_PAGES_FP4 : LTV_PAGES_VALUES,
                                k_pages.data_ptr(), kp.s, v_pages.data_ptr(), vp.s, &b.b,
                                k.data_ptr(), v.data_ptr(), (int)NKVH, (int)D, stream_of(k)),
           "ltv_paged_cache_read");
  return std::make_tuple(k, v);
}

// (compact needs no lengths)
ltv_page_state make_state(const Tensor& table, const OptTensor& lens, const Tensor& refs,
                          int page_size) {
  TORCH_CHECK(table.is_cuda(), "LTV HIP kernels need GPU tensors, got page_table on ",
              table.device());
  int_table(table, "page_table", 2, table);
  TORCH_CHECK_VALUE(rows_apart(table), "page_table's rows overlap, and are to be written");
  int_table(refs, "ref_counts", 1, table);
  ltv_page_state s{};
  if (lens.has_value()) {
    int_table(*lens, "seq_lens", 1, table);
    TORCH_CHECK_VALUE(lens->size(0) == table.size(0), "page_table has ", table.size(0),
                      " rows, seq_lens ", lens->size(0));
    s.seq_lens = lens->numel() ? lens->data_ptr<int32_t>() : nullptr;
  }
  s.page_table = table.numel() ? table.data_ptr<int32_t>() : nullptr;
  s.ref_counts = refs.numel() ? refs.data_ptr<int32_t>() : nullptr;
  s.table_stride = std::max(table.stride(0), table.size(1));
  s.num_slots = to_int(table.size(0), "the number of slots");
  s.table_width = to_int(table.size(1), "the page table's width");
  s.num_pages = to_int(refs.size(0), "the number of pages");
  s.page_size = page_size;
  return s;
}

// Pages of one layer (P, NKVH, page, D) or of all (layers, P, NKVH, page, D), each page
// one dense block in whatever order of its axes.
ltv_page_blocks make_blocks(const Tensor& k, const Tensor& v) {
  TORCH_CHECK(k.is_cuda(), "LTV HIP kernels need GPU tensors, got k_pages on ", k.device());
  on_device(v, "v_pages", k);
  TORCH_CHECK_VALUE((k.dim() == 4 || k.dim() == 5) && v.sizes() == k.sizes(),
                    "k_pages and v_pages must be ([layers,] pages, kv heads, page size, head_dim) "
                    "and alike, got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "k_pages are ", k.scalar_type(),
                   ", v_pages ", v.scalar_type());
  const int d0 = (int)k.dim() - 3;
  for (const Tensor* t : {&k, &v}) {
    // the strides of the block's axes, ascending, are the running products of the sizes
    int64_t want = 1;
    for (int i = 0; i < 3; ++i) {
      int at = -1;
      for (int d = d0; d < d0 + 3; ++d)
        if (t->size(d) > 1 && t->stride(d) == want) at = d;
      if (at < 0) break;
      want *= t->size(at);
    }
    TORCH_CHECK_VALUE(t->numel() == 0 || want == t->size(d0) * t->size(d0 + 1) * t->size(d0 + 2),
                      "each page must be a dense block of memory");
  }
  // (an axis of one element has no stride to speak of)
  for (int d = d0; d < d0 + 3; ++d)
    TORCH_CHECK_VALUE(k.numel() == 0 || k.size(d) == 1 || k.stride(d) == v.stride(d),
                      "k_pages and v_pages must be laid out alike");
  const int64_t es = k.element_size();
  auto bytes = [es](const Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d) * es; };
  ltv_page_blocks b{};
  b.k = k.data_ptr();
  b.v = v.data_ptr();
  b.k_page_bytes = bytes(k, d0 - 1);
  b.v_page_bytes = bytes(v, d0 - 1);
  b.layers = k.dim() == 5 ? to_int(k.size(0), "the number of layers") : 1;
  b.k_layer_bytes = k.dim() == 5 ? bytes(k, 0) : 0;
  b.v_layer_bytes = v.dim() == 5 ? bytes(v, 0) : 0;
  b.block_bytes = k.size(d0) * k.size(d0 + 1) * k.size(d0 + 2) * es;
  b.num_pages = to_int(k.size(d0 - 1), "the number of pages");
  return b;
}

OptTensor reserve(const Tensor& table, const Tensor& lens, const Tensor& refs,
                  const Tensor& slots_in, const Tensor& counts_in, const Tensor& k_pages,
                  const Tensor& v_pages) {
  if (!ordinary_call(table, lens, refs, slots_in, counts_in, k_pages, v_pages)) return {};
  const ltv_page_blocks blocks = make_blocks(k_pages, v_pages);
  on_device(table, "page_table", k_pages);
  const int page = to_int(k_pages.size(-2), "the page size");
  TORCH_CHECK_VALUE(page > 0, "a page must hold tokens");
  const ltv_page_state state = make_state(table, lens, refs, page);
  TORCH_CHECK_VALUE(blocks.num_pages == state.num_pages, blocks.num_pages, " pages, but ",
                    state.num_pages, " reference counts");
  const Tensor slots = int_vector(slots_in, "slots", table),
               counts = int_vector(counts_in, "counts", table);
  TORCH_CHECK_VALUE(slots.numel() == counts.numel(), slots.numel(), " slots, but ",
                    counts.numel(), " counts");
  c10::OptionalDeviceGuard guard(table.device());
  const int n = to_int(slots.numel(), "the number of slots");
  if (n == 0) return at::zeros({1}, table.options());
  Tensor status = at::empty({1}, table.options());
  const Workspace ws(ltv_paged_cache_reserve_workspace_size(n, state.num_pages));
  check_rc(ltv_paged_cache_reserve(&state, &blocks, slots.data_ptr<int32_t>(),
                                   counts.data_ptr<int32_t>(), n, status.data_ptr<int32_t>(),
                                   ws.ptr(), ws.bytes, stream_of(table)),
           "ltv_paged_cache_reserve");
  return status;
}

bool fork_slots(const Tensor& table, const Tensor& lens, const Tensor& refs, const Tensor& src_in,
                const Tensor& dst_in) {
  if (!ordinary_call(table, lens, refs, src_in, dst_in)) return false;
  const ltv_page_state state = make_state(table, lens, refs, 1);
  const Tensor src = int_vector(src_in, "src", table), dst = int_vector(dst_in, "dst", table);
  TORCH_CHECK_VALUE(src.numel() == dst.numel(), src.numel(), " src slots, but ", dst.numel(),
                    " dst slots");
  c10::OptionalDeviceGuard guard(table.device());
  if (src.numel() == 0) return true;
  check_rc(ltv_paged_cache_fork(&state, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(),
                                to_int(src.numel(), "the number of slots"), stream_of(table)),
           "ltv_paged_cache_fork");
  return true;
}

bool reorder_slots(const Tensor& table, const Tensor& lens, const Tensor& refs,
                   const Tensor& slots_in, const Tensor& src_in) {
  if (!ordinary_call(table, lens, refs, slots_in, src_in)) return false;
  const ltv_page_state state = make_state(table, lens, refs, 1);
  const Tensor slots = int_vector(slots_in, "slots", table), src = int_vector(src_in, "src", table);
  TORCH_CHECK_VALUE(slots.numel() == src.numel(), slots.numel(), " slots, but ", src.numel(),
                    " src slots");
  c10::OptionalDeviceGuard guard(table.device());
  if (slots.numel() == 0) return true;
  const int n = to_int(slots.numel(), "the number of slots");
  const Workspace ws(ltv_paged_cache_reorder_workspace_size(n, state.table_width));
  check_rc(ltv_paged_cache_reorder(&state, slots.data_ptr<int32_t>(), src.data_ptr<int32_t>(), n,
                                   ws.ptr(), ws.bytes, stream_of(table)),
           "ltv_paged_cache_reorder");
  return true;
}

bool free_slots(const Tensor& table, const Tensor& lens, const Tensor& refs,
                const Tensor& slots_in) {
  if (!ordinary_call(table, lens, refs, slots_in)) return false;
  const ltv_page_state state = make_state(table, lens, refs, 1);
  const Tensor slots = int_vector(slots_in, "slots", table);
  c10::OptionalDeviceGuard guard(table.device());
  if (slots.numel() == 0) return true;
  check_rc(ltv_paged_cache_free(&state, slots.data_ptr<int32_t>(),
                                to_int(slots.numel(), "the number of slots"), stream_of(table)),
           "ltv_paged_cache_free");
  return true;
}

bool copy_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& src_in,
                const Tensor& dst_in) {
  if (!ordinary_call(k_pages, v_pages, src_in, dst_in)) return false;
  const ltv_page_blocks blocks = make_blocks(k_pages, v_pages);
  const Tensor src = int_vector(src_in, "src", k_pages), dst = int_vector(dst_in, "dst", k_pages);
  TORCH_CHECK_VALUE(src.numel() == dst.numel(), src.numel(), " src pages, but ", dst.numel(),
                    " dst pages");
  c10::OptionalDeviceGuard guard(k_pages.device());
  if (src.numel() == 0) return true;
  check_rc(ltv_paged_cache_copy(&blocks, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(),
                                to_int(src.numel(), "the number of pages"), stream_of(k_pages)),
           "ltv_paged_cache_copy");
  return true;
}

OptTensor compact(const Tensor& table, const Tensor& refs, const Tensor& k_pages,
                  const Tensor& v_pages) {
  if (!ordinary_call(table, refs, k_pages, v_pages)) return {};
  const ltv_page_blocks blocks = make_blocks(k_pages, v_pages);
  on_device(table, "page_table", k_pages);
  ltv_page_state state = make_state(table, std::nullopt, refs, 1);
  TORCH_CHECK_VALUE(blocks.num_pages == state.num_pages, blocks.num_pages, " pages, but ",
                    state.num_pages, " reference counts");
  c10::OptionalDeviceGuard guard(table.device());
  Tensor live = at::empty({1}, table.options());
  const Workspace ws(ltv_paged_cache_compact_workspace_size(state.num_pages));
  check_rc(ltv_paged_cache_compact(&state, &blocks, live.data_ptr<int32_t>(), ws.ptr(), ws.bytes,
                                   stream_of(table)),
           "ltv_paged_cache_compact");
  return live;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// (out, lse or None)
std::optional<std::tuple<Tensor, OptTensor>> attention(
    const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table,
    const Tensor& lens, const OptTensor& slots, const OptTensor& starts, const OptInt& max_new,
    const OptInt& max_len, std::optional<double> scale, bool return_lse) {
  no_tangent(q_in, "q");
  no_tangent(k_pages, "k_pages");
  no_tangent(v_pages, "v_pages");
  if (!ordinary_call(q_in, k_pages, v_pages, table, lens, slots, starts)) return {};
  const int dt = dtype_of(q_in, "q");
  TORCH_CHECK(q_in.is_cuda(), "LTV HIP kernels need GPU tensors, got q on ", q_in.device());
  no_grad_needed(q_in, "q");
  check_any_pages(k_pages, v_pages, q_in);
  const Batch b = make_batch(q_in, "q", k_pages, table, lens, slots, starts, max_new);
  const int64_t NH = q_in.size(-2), D = q_in.size(-1), NKVH = k_pages.size(1);
  TORCH_CHECK_VALUE(head_dim_of(k_pages) == D, "q has head_dim ", D, ", the pages ",
                    head_dim_of(k_pages));
  TORCH_CHECK_VALUE(NH == 0 || (NKVH > 0 && NH % NKVH == 0), NKVH,
                    " k/v heads do not divide q's ", NH);
  TORCH_CHECK_VALUE(D > 0 && D <= 128 && D % 8 == 0,
                    "head_dim must be a multiple of 8, at most 128, got ", D);
  // (as the kernels have it, which multiply it by log2(e))
  const float sc = (float)scale.value_or(1.0 / std::sqrt((double)D));
  TORCH_CHECK_VALUE(std::isfinite(sc * 1.4427f) && sc > 0,
                    "scale must be positive and finite in float32, got ", scale.value_or(sc));
  const int most = to_int(std::min<int64_t>(max_len.value_or(table.size(1) * k_pages.size(2)),
                                            table.size(1) * k_pages.size(2)),
                          "max_len");
  const Tensor q = rows_contiguous(q_in);
  c10::OptionalDeviceGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
  OptTensor lse;
  if (return_lse) lse = at::empty(q.sizes().slice(0, q.dim() - 1), out.options().dtype(at::kFloat));
  if (out.numel() == 0) return std::make_tuple(out, lse);
  const bool fp4 = is_fp4(k_pages);
  const Workspace ws((fp4 ? ltv_paged_attention_fp4_workspace_size
                          : ltv_paged_attention_workspace_size)(dt, &b.b, (int)NH, (int)NKVH,
                                                                (int)D, most));
  const Strides3 qs = Strides3::tokens(q), os = Strides3::tokens(out),
                 kp = any_strides(k_pages), vp = any_strides(v_pages);
  check_rc((fp4 ? ltv_paged_attention_fp4 : ltv_paged_attention)(
               dt, q.data_ptr(), qs.s, k_pages.data_ptr(), kp.s, v_pages.data_ptr(), vp.s, &b.b,
               out.data_ptr(), os.s, lse.has_value() ? lse->data_ptr<float>() : nullptr, ws.ptr(),
               ws.bytes, (int)NH, (int)NKVH, (int)D, most, sc, stream_of(q)),
           fp4 ? "ltv_paged_attention_fp4" : "ltv_paged_attention");
  return std::make_tuple(out, lse);
}

// ---------------------------------------------------------------------------
// log probabilities
// ---------------------------------------------------------------------------
struct Rows {
  Tensor x, targets;  // (N, V), (N)
};

Rows rows_of(const Tensor& logits, const Tensor& targets) {
  dtype_of(logits, "logits");
  TORCH_CHECK(logits.is_cuda(), "LTV HIP kernels need GPU tensors, got logits on ",
              logits.device());
  on_device(targets, "targets", logits);
  TORCH_CHECK_VALUE(logits.dim() >= 1 &&
                        targets.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "logits must be (..., vocabulary) and targets (...), got ", logits.sizes(),
                    " and ", targets.sizes());
  TORCH_CHECK_TYPE(targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt,
                   "targets must be int64 or int32, got ", targets.scalar_type());
  TORCH_CHECK_VALUE(logits.size(-1) > 0, "an empty vocabulary");
  Rows r;
  r.x = logits.dim() == 2 ? logits : logits.reshape({targets.numel(), logits.size(-1)});
  if (r.x.size(1) > 1 && r.x.stride(1) != 1) r.x = r.x.contiguous();
  r.targets = targets.reshape({targets.numel()});
  if (r.targets.scalar_type() != at::kLong) r.targets = r.targets.to(at::kLong);
  r.targets = r.targets.contiguous();
  return r;
}

struct LogpOut {
  Tensor logprobs, entropy, top, ids, lse;
};

LogpOut logprobs_forward(const Tensor& logits, const Tensor& targets, int64_t top_k, double cap,
                         bool keep_lse) {
  const Rows r = rows_of(logits, targets);
  const int64_t N = r.x.size(0), V = r.x.size(1);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= 64 && top_k <= V,
                    "top_k must be 0 to 64 and no more than the vocabulary of ", V, ", got ",
                    top_k);
  TORCH_CHECK_VALUE(std::isfinite((float)cap) && cap >= 0 && ((float)cap > 0 || cap == 0),
                    "softcap must be positive and finite in float32, got ", cap);
  c10::OptionalDeviceGuard guard(r.x.device());
  const auto f32 = r.x.options().dtype(at::kFloat).requires_grad(false);
  const auto shape = targets.sizes().vec();
  auto top_shape = shape;
  top_shape.push_back(top_k);
  LogpOut o{at::empty(shape, f32), at::empty(shape, f32), at::empty(top_shape, f32),
            at::empty(top_shape, f32.dtype(at::kLong)), keep_lse ? at::empty(shape, f32) : Tensor()};
  if (N == 0) return o;
  const Workspace ws(
      ltv_token_logprobs_workspace_size(N, to_int(V, "the vocabulary"), (int)top_k));
  check_rc(ltv_token_logprobs_forward(
               dtype_of(r.x, "logits"), r.x.data_ptr(), r.x.stride(0),
               r.targets.data_ptr<int64_t>(), o.logprobs.data_ptr<float>(),
               o.entropy.data_ptr<float>(), keep_lse ? o.lse.data_ptr<float>() : nullptr,
               top_k > 0 ? o.top.data_ptr<float>() : nullptr,
               top_k > 0 ? o.ids.data_ptr<int64_t>() : nullptr, ws.ptr(), ws.bytes, N, (int)V,
               (int)top_k, (float)cap, stream_of(r.x)),
           "ltv_token_logprobs_forward");
  return o;
}

Tensor backward_of(const Tensor& logits, const Tensor& targets, const Tensor& lse,
                   const Tensor& entropy, const Tensor& ids, const OptTensor& g_lp,
                   const OptTensor& g_ent, const OptTensor& g_top, double cap) {
  no_tangent(logits, "logits");
  const Rows r = rows_of(logits, targets);
  c10::OptionalDeviceGuard guard(r.x.device());
  Tensor gx = at::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(
                                            at::MemoryFormat::Contiguous));
  if (gx.numel() == 0) return gx;
  auto grad = [](const OptTensor& g) {
    if (!g.has_value() || !g->defined()) return Tensor();
    no_tangent(*g, "the gradient");
    return g->to(at::kFloat).contiguous();
  };
  auto ptr = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  const Tensor a = grad(g_lp), b = grad(g_ent), c = grad(g_top);
  const int64_t V = r.x.size(1), k = ids.size(-1);
  const Tensor le = lse.contiguous(), en = entropy.contiguous(), id = ids.contiguous();
  check_rc(ltv_token_logprobs_backward(
               dtype_of(r.x, "logits"), r.x.data_ptr(), r.x.stride(0),
               r.targets.data_ptr<int64_t>(), le.data_ptr<float>(), en.data_ptr<float>(),
               k > 0 ? id.data_ptr<int64_t>() : nullptr, ptr(a), ptr(b), k > 0 ? ptr(c) : nullptr,
               gx.data_ptr(), V, r.x.size(0), (int)V, (int)k, (float)cap, stream_of(r.x)),
           "ltv_token_logprobs_backward");
  return gx;
}

class TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets,
                               int64_t top_k, double cap) {
    LogpOut o = logprobs_forward(logits, targets, top_k, cap, true);
    ctx->save_for_backward({logits, targets, o.lse, o.entropy, o.ids});
    ctx->saved_data["cap"] = cap;
    ctx->mark_non_differentiable({o.ids});
    ctx->set_materialize_grads(false);
    return {o.logprobs, o.entropy, o.top, o.ids};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const variable_list s = ctx->get_saved_variables();
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return {{}, {}, {}, {}};
    Tensor gx = backward_of(s[0], s[1], s[2], s[3], s[4], g[0], g[1], g[2],
                            ctx->saved_data["cap"].toDouble());
    // (with create_graph: a second derivative is refused, not taken as zero)
    if (at::GradMode::is_enabled())
      torch::autograd::set_history(
          gx, std::make_shared<torch::autograd::Error>(
                  "token_logprobs is differentiable once only",
                  torch::autograd::collect_next_edges(s[0], g[0], g[1], g[2])));
    return {gx, {}, {}, {}};
  }
};

// (logprobs, entropy, top_logprobs, top_ids)
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> token_logprobs(const Tensor& logits,
                                                                         const Tensor& targets,
                                                                         int64_t top_k,
                                                                         double cap) {
  no_tangent(logits, "logits");
  if (!ordinary_call(logits, targets)) return {};
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list o = TokenLogprobs::apply(logits, targets, top_k, cap);
    return std::make_tuple(o[0], o[1], o[2], o[3]);
  }
  LogpOut o = logprobs_forward(logits, targets, top_k, cap, false);
  return std::make_tuple(o.logprobs, o.entropy, o.top, o.ids);
}

// (with the row sums that the backward reads)
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>> token_logprobs_forward(
    const Tensor& logits, const Tensor& targets, int64_t top_k, double cap) {
  no_tangent(logits, "logits");
  if (!ordinary_call(logits, targets)) return {};
  LogpOut o = logprobs_forward(logits, targets, top_k, cap, true);
  return std::make_tuple(o.logprobs, o.entropy, o.top, o.ids, o.lse);
}

OptTensor token_logprobs_backward(const Tensor& logits, const Tensor& targets, const Tensor& lse,
                                  const Tensor& entropy, const Tensor& ids, const OptTensor& g_lp,
                                  const OptTensor& g_ent, const OptTensor& g_top, double cap) {
  if (!ordinary_call(logits, targets, lse, entropy, ids, g_lp, g_ent, g_top)) return {};
  return backward_of(logits, targets, lse, entropy, ids, g_lp, g_ent, g_top, cap);
}

// ---------------------------------------------------------------------------
// a search's selection
// ---------------------------------------------------------------------------
// (scores, parents, tokens)
std::optional<std::tuple<Tensor, Tensor, Tensor>> beam_select(const Tensor& logits,
                                                              const Tensor& scores_in, int64_t k,
                                                              double cap,
                                                              const OptTensor& finished_in) {
  no_tangent(logits, "logits");
  no_tangent(scores_in, "scores");
  if (!ordinary_call(logits, scores_in, finished_in)) return {};
  const int dt = dtype_of(logits, "logits");
  TORCH_CHECK(logits.is_cuda(), "LTV HIP kernels need GPU tensors, got logits on ",
              logits.device());
  on_device(scores_in, "scores", logits);
  const auto no_grad = [](const Tensor& t, const char* name) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
                " requires grad, but a selection has none: call under torch.no_grad()");
  };
  no_grad(logits, "logits");
  no_grad(scores_in, "scores");
  TORCH_CHECK_VALUE(logits.dim() >= 2 &&
                        scores_in.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "logits must be (..., beams, vocabulary) and scores (..., beams), got ",
                    logits.sizes(), " and ", scores_in.sizes());
  TORCH_CHECK_TYPE(scores_in.scalar_type() == at::kFloat, "scores must be float32, got ",
                   scores_in.scalar_type());
  const int64_t B = logits.size(-2), V = logits.size(-1);
  TORCH_CHECK_VALUE(B > 0 && V > 0, "no beams, or an empty vocabulary: ", logits.sizes());
  TORCH_CHECK_VALUE(k > 0 && (k - 1) / B < V, "k must be 1 to the ", B, " beams' tokens, got ", k);
  const int64_t n = std::min(k, V);
  TORCH_CHECK_VALUE(n <= 64 && B * n <= 1024, "at most 64 continuations of a beam and 1,024 of all, "
                    "got k ", k, " of ", B, " beams");
  TORCH_CHECK_VALUE(std::isfinite((float)cap) && cap >= 0 && ((float)cap > 0 || cap == 0),
                    "softcap must be positive and finite in float32, got ", cap);
  Tensor finished;
  if (finished_in.has_value()) {
    on_device(*finished_in, "finished", logits);
    TORCH_CHECK_TYPE(finished_in->scalar_type() == at::kBool, "finished must be bool, got ",
                     finished_in->scalar_type());
    TORCH_CHECK_VALUE(finished_in->sizes() == scores_in.sizes(), "scores is ", scores_in.sizes(),
                      ", finished ", finished_in->sizes());
    finished = finished_in->contiguous();
  }
  c10::OptionalDeviceGuard guard(logits.device());
  const int64_t G = scores_in.numel() / B;
  Tensor x = logits.reshape({G * B, V});
  if (V > 1 && x.stride(1) != 1) x = x.contiguous();
  const Tensor scores = scores_in.contiguous();
  auto shape = scores_in.sizes().vec();
  shape.back() = k;
  const auto f32 = scores.options().requires_grad(false);
  Tensor best = at::empty(shape, f32), parents = at::empty(shape, f32.dtype(at::kLong)),
         tokens = at::empty(shape, f32.dtype(at::kLong));
  if (G == 0) return std::make_tuple(best, parents, tokens);
  const int b = to_int(B, "the number of beams"), v = to_int(V, "the vocabulary"),
            kk = to_int(k, "k");
  const Workspace ws(ltv_beam_select_workspace_size(G, b, v, kk));
  check_rc(ltv_beam_select(dt, x.data_ptr(), x.stride(0), scores.data_ptr<float>(),
                           finished.defined()
                               ? reinterpret_cast<const uint8_t*>(finished.data_ptr<bool>())
                               : nullptr,
                           best.data_ptr<float>(), parents.data_ptr<int64_t>(),
                           tokens.data_ptr<int64_t>(), ws.ptr(), ws.bytes, G, b, v, kk, (float)cap,
                           stream_of(x)),
           "ltv_beam_select");
  return std::make_tuple(best, parents, tokens);
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  using nogil = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("paged_cache_append", &append, nogil());
  m.def("paged_rotary_append", &rotary_append, nogil());
  m.def("paged_cache_read", &read_pages, nogil());
  m.def("paged_cache_reorder", &reorder_slots, nogil());
  m.def("paged_cache_reserve", &reserve, nogil());
  m.def("paged_cache_fork", &fork_slots, nogil());
  m.def("paged_cache_free", &free_slots, nogil());
  m.def("paged_cache_copy", &copy_pages, nogil());
  m.def("paged_cache_compact", &compact, nogil());
  m.def("paged_attention", &attention, nogil());
  m.def("beam_select", &beam_select, nogil());
  m.def("token_logprobs", &token_logprobs, nogil());
  m.def("token_logprobs_forward", &token_logprobs_forward, nogil());
  m.def("token_logprobs_backward", &token_logprobs_backward, nogil());
}
