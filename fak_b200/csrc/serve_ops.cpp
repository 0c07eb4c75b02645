// Torch entry points of the 4-bit KV cache, batch plan and log-probability kernels: argument checks and
// launches on the current stream of the inputs' device.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>

#include <cmath>
#include <map>
#include <mutex>

#include "serve_ops.h"

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

// Numbers in messages: formatted without iostreams (an extension linked against a static C++ runtime
// cannot stream a number into a message: its locale facets are not those of torch's libraries).
std::string S(int64_t v) { return std::to_string(v); }

fak::Elt elt(const Tensor& t, const char* what) {
  if (t.scalar_type() == torch::kFloat32) return fak::Elt::F32;
  if (t.scalar_type() == torch::kFloat16) return fak::Elt::F16;
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, what, ": want float32, float16 or bfloat16, got ", c10::toString(t.scalar_type()));
  return fak::Elt::BF16;
}
int* err_ptr(const OptTensor& err, const Tensor& like) {
  if (!err.has_value()) return nullptr;
  TORCH_CHECK(err->scalar_type() == torch::kInt32 && err->numel() >= 1 && err->device() == like.device(),
              "err: int32 word on the inputs' device");
  return err->data_ptr<int>();
}
const int* i32(const Tensor& t, int64_t n, const Tensor& like, const char* what) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.is_contiguous() &&
                  t.numel() >= n, what, ": want a contiguous int32 vector of at least ", S(n), " on the inputs' device");
  return t.data_ptr<int>();
}
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()); }
int sms(const Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

// the layer's pages [P, Hkv, 20 D]: returns D
int check_pages(const Tensor& pages, const char* what) {
  TORCH_CHECK(pages.is_cuda() && pages.scalar_type() == torch::kUInt8 && pages.dim() == 3 && pages.is_contiguous(), what,
              ": pages are a contiguous uint8 [pages, kv heads, bytes] CUDA tensor");
  TORCH_CHECK(pages.size(2) == 1280 || pages.size(2) == 2560, what, ": ", S(pages.size(2)),
              " bytes per page and head: head dim must be 64 (1280) or 128 (2560)");
  TORCH_CHECK(pages.size(0) > 0 && pages.size(1) > 0, what, ": no pages");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0, what, ": pages must start on a 16-byte boundary");
  return (int)pages.size(2) / 20;
}
// A tensor inside a buffer of its own type: the parts of a plan share one allocation.
Tensor carve(const Tensor& buf, int64_t at, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}
int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }
// Zeroed counters, left at zero by every launch: one set per stream, so that calls on different streams
// cannot meet in them.  A captured call gets its own, which the graph zeroes.
Tensor tickets_for(const Tensor& like, int64_t n) {
  auto opt = like.options().dtype(torch::kInt32);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return torch::zeros({n}, opt);
  static std::mutex mu;
  static auto* held = new std::map<std::pair<int, cudaStream_t>, Tensor>();   // (lives as long as the process)
  std::lock_guard<std::mutex> lock(mu);
  Tensor& t = (*held)[{like.get_device(), stream_of(like)}];
  if (!t.defined() || t.numel() < n) t = torch::zeros({std::max<int64_t>(n, 4096)}, opt);
  return t;
}
// Some of v's first n elements lie among `rows` rows of `width` elements, `stride` apart, at t (4-byte elements).
bool meets(const Tensor& v, int64_t n, const Tensor& t, int64_t rows, int64_t width, int64_t stride) {
  if (n == 0 || rows == 0 || width == 0) return false;
  const int64_t at = ((intptr_t)v.data_ptr() - (intptr_t)t.data_ptr()) / 4;
  const int64_t row = stride > 0 && at >= width ? (at - width) / stride + 1 : 0;   // the first that ends past v's start
  return row < rows && row * stride < at + n && row * stride + width > at;
}
// rows (of a tensor that may be expanded) as the kernels count them
int rows32(int64_t n, const char* what) {
  TORCH_CHECK(n <= INT32_MAX, what, ": ", S(n), " rows are too many");
  return (int)n;
}
bool aligned(const Tensor& t, int64_t elems) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % (elems * t.element_size()) == 0;
}

}  // namespace

void kv4_append(Tensor k, Tensor v, Tensor slot, Tensor pages, OptTensor err) {
  const int D = check_pages(pages, "kv4_append");
  const int64_t Hkv = pages.size(1);
  fak::Kv4Rows r{};
  r.type = elt(k, "kv4_append: k");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), "kv4_append: k and v differ in type");
  const int64_t T = rows32(slot.numel(), "kv4_append");
  r.vec = true;
  auto rows = [&](const Tensor& x, const char* what, int64_t& s_page, int64_t& s_row, int64_t& s_head) {
    TORCH_CHECK(x.device() == pages.device(), "kv4_append: ", what, " is not on the pages' device");
    TORCH_CHECK(x.dim() == 3 || x.dim() == 4, "kv4_append: ", what, " is [T, kv heads, D] or bf16-cache pages [P, kv heads, 16, D]");
    const int hd = (int)x.dim() - 2 - (x.dim() == 4 ? 1 : 0);
    TORCH_CHECK(x.size(-1) == D && x.size(hd) == Hkv, "kv4_append: ", what, " has ", S(x.size(hd)), " heads of ", S(x.size(-1)),
                ", the pages ", S(Hkv), " of ", S(D));
    TORCH_CHECK(x.stride(-1) == 1 || D == 1, "kv4_append: ", what, "'s last dimension must be contiguous");
    if (x.dim() == 4) {
      TORCH_CHECK(x.size(2) == 16 && x.size(0) * 16 >= T, "kv4_append: ", what, " pages hold fewer than ", S(T), " tokens");
      s_page = x.stride(0);
      s_row = x.stride(2);
      s_head = x.stride(1);
    } else {
      TORCH_CHECK(x.size(0) == T, "kv4_append: ", what, " has ", S(x.size(0)), " rows for ", S(T), " slots");
      s_row = x.stride(0);
      s_page = 16 * s_row;
      s_head = x.stride(1);
    }
    const int64_t per = fak::kKv4LoadBytes / x.element_size();
    r.vec = r.vec && aligned(x, per) && s_page % per == 0 && s_row % per == 0 && s_head % per == 0;
  };
  rows(k, "k", r.ks_page, r.ks_row, r.ks_head);
  rows(v, "v", r.vs_page, r.vs_row, r.vs_head);
  const int* sl = i32(slot, T, pages, "kv4_append: slot");
  TORCH_CHECK(T * Hkv < (int64_t(1) << 33), "kv4_append: too many rows");
  c10::cuda::CUDAGuard guard(pages.device());
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  fak::kv4_append_launch(r, sl, (int)T, (int)Hkv, D, pages.data_ptr<uint8_t>(), pages.size(0), err_ptr(err, pages),
                         stream_of(pages));
}

std::vector<Tensor> kv4_read(Tensor pages, Tensor slot, int64_t head_dim, c10::ScalarType dtype, OptTensor err) {
  const int D = check_pages(pages, "kv4_read");
  TORCH_CHECK(D == head_dim, "kv4_read: the pages hold heads of ", S(D), ", not ", S(head_dim));
  const int64_t T = rows32(slot.numel(), "kv4_read"), Hkv = pages.size(1);
  const int* sl = i32(slot, T, pages, "kv4_read: slot");
  c10::cuda::CUDAGuard guard(pages.device());
  auto opt = pages.options().dtype(dtype);
  Tensor k = torch::empty({T, Hkv, D}, opt), v = torch::empty({T, Hkv, D}, opt);
  fak::kv4_read_launch(pages.data_ptr<uint8_t>(), pages.size(0), sl, (int)T, (int)Hkv, D, k.data_ptr(), v.data_ptr(),
                       elt(k, "kv4_read: dtype"), err_ptr(err, pages), stream_of(pages));
  return {k, v};
}

void kv4_attention(Tensor q, Tensor pages, Tensor table, OptTensor q_off, Tensor ctx, Tensor out, int64_t max_new,
                   double scale, double softcap, int64_t window, OptTensor sinks, int64_t n_split, OptTensor workspace,
                   OptTensor err, int64_t tiles) {
  fak::Kv4Attn a{};
  a.D = check_pages(pages, "kv4_attention");
  a.Hkv = (int)pages.size(1);
  TORCH_CHECK(q.device() == pages.device() && q.dim() == 3 && q.size(2) == a.D && q.stride(2) == 1,
              "kv4_attention: q is [T, heads, ", S(a.D), "] on the pages' device, last dimension contiguous");
  TORCH_CHECK(q.size(1) > 0 && q.size(1) % a.Hkv == 0, "kv4_attention: ", S(q.size(1)), " query heads over ", S(a.Hkv), " kv heads");
  TORCH_CHECK(out.device() == q.device() && out.sizes() == q.sizes() && out.stride(2) == 1,
              "kv4_attention: out has q's shape, last dimension contiguous");
  TORCH_CHECK(table.device() == q.device() && table.scalar_type() == torch::kInt32 && table.dim() == 2 && table.stride(1) == 1,
              "kv4_attention: block table int32 [B, W]");
  a.q = q.data_ptr();
  a.q_type = elt(q, "kv4_attention: q");
  a.q_tok = q.stride(0);
  a.q_head = q.stride(1);
  a.q_vec = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_tok * q.element_size() % 16 == 0 && a.q_head * q.element_size() % 16 == 0;
  a.out = out.data_ptr();
  a.o_type = elt(out, "kv4_attention: out");
  a.o_tok = out.stride(0);
  a.o_head = out.stride(1);
  a.o_vec = out.element_size() == 2 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.o_tok % 8 == 0 && a.o_head % 8 == 0;
  a.pages = pages.data_ptr<uint8_t>();
  a.n_pages = pages.size(0);
  a.table = table.data_ptr<int>();
  a.table_stride = table.stride(0);
  a.width = (int)std::min<int64_t>(table.size(1), INT32_MAX / 16);
  a.n_tokens = rows32(q.size(0), "kv4_attention");
  a.ctx = i32(ctx, 0, q, "kv4_attention: ctx_len");
  a.H = (int)q.size(1);
  a.G = a.H / a.Hkv;
  a.g_inv = a.G > 1 ? (uint32_t)(((uint64_t(1) << 32) + a.G - 1) / a.G) : 0;
  a.B = rows32(ctx.numel(), "kv4_attention");
  a.max_new = (int)max_new;
  TORCH_CHECK(table.size(0) >= a.B, "kv4_attention: block table has ", S(table.size(0)), " rows for ", S(a.B), " sequences");
  if (q_off.has_value()) {
    a.q_off = i32(*q_off, a.B + 1, q, "kv4_attention: q_off");
    TORCH_CHECK(max_new >= 0 && max_new <= q.size(0), "kv4_attention: max_new ", S(max_new), " outside [0, ", S(q.size(0)), "]");
  } else {
    TORCH_CHECK(a.B == a.n_tokens && max_new == 1, "kv4_attention: ", S(a.n_tokens), " queries for ", S(a.B), " sequences");
  }
  if (sinks.has_value()) {
    TORCH_CHECK(sinks->device() == q.device() && sinks->scalar_type() == torch::kFloat32 && sinks->is_contiguous() &&
                    sinks->numel() >= a.H, "kv4_attention: sinks [H] float32");
    a.sinks = sinks->data_ptr<float>();
  }
  TORCH_CHECK(softcap >= 0 && std::isfinite((float)softcap), "kv4_attention: softcap ", std::to_string(softcap), " (0: none)");
  TORCH_CHECK(n_split >= 0 && n_split <= 4096, "kv4_attention: n_split in [0, 4096]");
  TORCH_CHECK(scale >= 0 && std::isfinite((float)scale), "kv4_attention: scale ", std::to_string(scale), " (0: 1 / sqrt of the head dim)");
  a.scale = scale > 0 ? (float)scale : 1.0f / std::sqrt((float)a.D);
  a.softcap = (float)softcap;
  a.window = (int)std::min<int64_t>(std::max<int64_t>(window, 0), INT32_MAX);   // (contexts are 32-bit)
  a.n_split = (int)n_split;
  a.tiles = (int)tiles;
  a.err = err_ptr(err, q);
  TORCH_CHECK(a.B <= 65535 && a.Hkv <= 65535, "kv4_attention: at most 65535 sequences and kv heads");
  TORCH_CHECK((int64_t)a.max_new * a.G < (int64_t(1) << 32) / a.G, "kv4_attention: too many query rows");
  if (a.B == 0 || a.n_tokens == 0 || a.max_new == 0) return;
  c10::cuda::CUDAGuard guard(q.device());
  const fak::Kv4AttnPlan p = fak::kv4_attn_plan(a, sms(q));
  TORCH_CHECK((int64_t)a.B * a.Hkv * p.row_chunks * std::max(p.n_split, 32) < (int64_t(1) << 31), "kv4_attention: too many query rows");
  Tensor ws;
  if (p.part_floats > 0) {
    if (workspace.has_value()) {
      TORCH_CHECK(workspace->device() == q.device() && workspace->scalar_type() == torch::kFloat32 &&
                      workspace->is_contiguous() && workspace->numel() >= p.part_floats && aligned(*workspace, 4),
                  "kv4_attention: workspace of at least ", S(p.part_floats), " float32");
      ws = *workspace;
    } else {
      ws = torch::empty({p.part_floats}, q.options().dtype(torch::kFloat32));
    }
    a.part = ws.data_ptr<float>();
  }
  fak::kv4_attn_launch(a, p, stream_of(q));
}

std::vector<Tensor> plan_batch(Tensor old_len, Tensor new_len, Tensor table, Tensor free_pages, Tensor free_head,
                               int64_t max_tokens, c10::optional<std::vector<Tensor>> outs, OptTensor err) {
  TORCH_CHECK(old_len.is_cuda(), "plan_batch: lengths are CUDA tensors");
  fak::BatchPlanArgs a{};
  const int64_t B = old_len.numel();
  TORCH_CHECK(B <= 16384, "plan_batch: at most 16384 requests, got ", S(B));
  TORCH_CHECK(new_len.numel() == B, "plan_batch: ", S(B), " cached lengths and ", S(new_len.numel()), " new ones");
  TORCH_CHECK(max_tokens >= 0 && max_tokens < (int64_t(1) << 30), "plan_batch: max_tokens ", S(max_tokens));
  a.old_len = i32(old_len, B, old_len, "plan_batch: cached lengths");
  a.new_len = i32(new_len, B, old_len, "plan_batch: new lengths");
  TORCH_CHECK(table.device() == old_len.device() && table.scalar_type() == torch::kInt32 && table.dim() == 2 &&
                  (table.stride(1) == 1 || table.size(1) <= 1) && table.size(0) >= B, "plan_batch: block table int32 [>= ", S(B), ", W]");
  a.B = (int)B;
  a.table = table.data_ptr<int>();
  a.table_stride = table.stride(0);
  a.width = (int)std::min<int64_t>(table.size(1), INT32_MAX / 16 + 1);
  a.n_free = rows32(free_pages.numel(), "plan_batch: free pages");
  a.free_pages = i32(free_pages, 0, old_len, "plan_batch: free pages");
  a.head = i32(free_head, 1, old_len, "plan_batch: free head");
  a.max_tokens = (int)max_tokens;
  a.err = err_ptr(err, old_len);
  c10::cuda::CUDAGuard guard(old_len.device());
  std::vector<Tensor> o;
  if (outs.has_value()) {
    o = *outs;
    TORCH_CHECK(o.size() == 7, "plan_batch: a plan has 7 tensors");
    const int64_t n[7] = {max_tokens, max_tokens, max_tokens, B + 1, B, B, 1};
    for (int i = 0; i < 7; i++) i32(o[i], n[i], old_len, "plan_batch: plan tensor");
    TORCH_CHECK(o[6].data_ptr() != free_head.data_ptr(), "plan_batch: the new free head needs a word of its own");
    // CTAs read the lengths, the table and the free pages while others write the plan
    for (int i = 0; i < 7; i++) {
      for (const Tensor* in : {&old_len, &new_len, &free_pages, &free_head})
        TORCH_CHECK(!meets(o[i], n[i], *in, 1, in->numel(), 0), "plan_batch: a plan tensor shares memory with the lengths or free pages");
      TORCH_CHECK(!meets(o[i], n[i], table, table.size(0), table.size(1), table.stride(0)), "plan_batch: a plan tensor shares memory with the block table");
      for (int j = 0; j < i; j++) TORCH_CHECK(!meets(o[i], n[i], o[j], 1, n[j], 0), "plan_batch: plan tensors share memory");
    }
  } else {
    const int64_t n[7] = {max_tokens, max_tokens, max_tokens, B + 1, B, B, 1};
    int64_t at = 0, all = 0;
    for (int64_t k : n) all += up4(k);
    Tensor buf = torch::empty({all}, old_len.options());
    o.reserve(7);
    for (int64_t k : n) {
      o.push_back(carve(buf, at, {k}));
      at += up4(k);
    }
  }
  a.slot = o[0].data_ptr<int>();
  a.pos = o[1].data_ptr<int>();
  a.seq = o[2].data_ptr<int>();
  a.q_off = o[3].data_ptr<int>();
  a.ctx = o[4].data_ptr<int>();
  a.last = o[5].data_ptr<int>();
  a.head_out = o[6].data_ptr<int>();
  fak::batch_plan_launch(a, stream_of(old_len));
  return o;
}

std::vector<Tensor> token_logprobs(Tensor logits, int64_t V, Tensor target, int64_t k, double softcap) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) <= 1),
              "token_logprobs: logits [T, >= V] on the GPU, last dimension contiguous");
  TORCH_CHECK(V > 0 && V <= logits.size(1) && V < (int64_t(1) << 30), "token_logprobs: V ", S(V), " of ", S(logits.size(1)), " columns");
  TORCH_CHECK(k >= 0 && k <= 32, "token_logprobs: 0 to 32 alternatives, got ", S(k));
  TORCH_CHECK(softcap >= 0 && std::isfinite((float)softcap), "token_logprobs: softcap ", std::to_string(softcap), " (0: none)");
  fak::LogprobArgs a{};
  a.type = elt(logits, "token_logprobs: logits");
  a.T = rows32(logits.size(0), "token_logprobs");
  a.V = (int)V;
  a.k = (int)k;
  a.x = logits.data_ptr();
  a.stride = logits.stride(0);
  a.target = i32(target, a.T, logits, "token_logprobs: targets");
  a.softcap = (float)softcap;
  const int64_t per = a.type == fak::Elt::F32 ? 4 : 8;
  a.vec = aligned(logits, per) && (a.stride % per == 0 || a.T <= 1);
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t T = a.T;
  const auto f32 = logits.options().dtype(torch::kFloat32), i32t = logits.options().dtype(torch::kInt32);
  Tensor lp = torch::empty({T}, f32), en = torch::empty({T}, f32), rank = torch::empty({T}, i32t);
  Tensor ids = torch::empty({T, k}, i32t), top = torch::empty({T, k}, f32);
  a.logprob = lp.data_ptr<float>();
  a.entropy = en.data_ptr<float>();
  a.rank = rank.data_ptr<int>();
  a.top_ids = ids.data_ptr<int>();
  a.top_logprobs = top.data_ptr<float>();
  if (T == 0) return {lp, en, rank, ids, top};
  a.n_seg = fak::logprob_segments(a.T, a.V, sms(logits));
  Tensor part, tickets;
  if (a.n_seg > 1) {
    tickets = tickets_for(logits, T);
    a.tickets = tickets.data_ptr<int>();
    part = torch::empty({fak::logprob_part_words(a.T, a.n_seg)}, f32);
    a.part = part.data_ptr<float>();
  }
  fak::logprob_launch(a, stream_of(logits));
  return {lp, en, rank, ids, top};
}

void bind_serve_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("kv4_append", &kv4_append, py::arg("k"), py::arg("v"), py::arg("slot"), py::arg("pages"), py::arg("err") = py::none());
  m.def("kv4_read", &kv4_read, py::arg("pages"), py::arg("slot"), py::arg("head_dim"), py::arg("dtype"),
        py::arg("err") = py::none());
  m.def("kv4_attention", &kv4_attention, py::arg("q"), py::arg("pages"), py::arg("table"), py::arg("q_off"), py::arg("ctx"),
        py::arg("out"), py::arg("max_new"), py::arg("scale") = 0.0, py::arg("softcap") = 0.0, py::arg("window") = 0,
        py::arg("sinks") = py::none(), py::arg("n_split") = 0, py::arg("workspace") = py::none(),
        py::arg("err") = py::none(), py::arg("tiles") = -1);
  m.def("plan_batch", &plan_batch, py::arg("old_len"), py::arg("new_len"), py::arg("table"), py::arg("free_pages"),
        py::arg("free_head"), py::arg("max_tokens"), py::arg("outs") = py::none(), py::arg("err") = py::none());
  m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("V"), py::arg("target"), py::arg("k"),
        py::arg("softcap") = 0.0);
}
