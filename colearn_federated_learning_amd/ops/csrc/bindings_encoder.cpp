// Python bindings of the encoder-training kernels: masked attention, residual
// add + layer norm, AdamW over many tensors.  Everything a kernel assumes of
// its operands is checked here, before a launch.

#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <utility>
#include <vector>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "encoder_api.h"

#define HIP_CHECK_LAST()                                          \
  do {                                                            \
    hipError_t e_ = hipGetLastError();                            \
    TORCH_CHECK(e_ == hipSuccess, "HIP kernel launch failed: ",   \
                hipGetErrorString(e_));                           \
  } while (0)

namespace colearn {

namespace {

// a launch has fewer than 2^32 threads
constexpr int64_t kMostThreads = std::numeric_limits<uint32_t>::max();
constexpr int64_t kMostBlocks = kMostThreads / 256;  // of 256 threads

using OptTensor = std::optional<torch::Tensor>;

hipStream_t stream() {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

Elem elem_of(const torch::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32:
      return Elem::kF32;
    case torch::kBFloat16:
      return Elem::kBF16;
    case torch::kFloat16:
      return Elem::kF16;
    default:
      TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, not ",
                  t.scalar_type());
  }
}

void check_gpu(const torch::Tensor& t, const torch::Device& dev,
               const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name,
              " must be on the GPU of the first operand (", dev, "), not ",
              t.device());
}

void check_like(const torch::Tensor& t, const torch::Tensor& like,
                const char* name) {
  check_gpu(t, like.device(), name);
  TORCH_CHECK(t.scalar_type() == like.scalar_type() &&
                  t.sizes() == like.sizes(),
              name, " must have the type and shape of the first operand");
}

bool aligned16(const torch::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// no byte of either contiguous tensor is the other's
bool apart(const torch::Tensor& a, const torch::Tensor& b) {
  const auto at = [](const torch::Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr());
  };
  return at(a) + a.nbytes() <= at(b) || at(b) + b.nbytes() <= at(a);
}

// ---- AdamW ------------------------------------------------------------------
void adamw_step(std::vector<torch::Tensor> p, std::vector<torch::Tensor> g,
                std::vector<torch::Tensor> m, std::vector<torch::Tensor> v,
                std::vector<torch::Tensor> ms, std::vector<torch::Tensor> vs,
                std::vector<torch::Tensor> ref, std::vector<double> keep,
                double b1, double b2, double eps, double mu, double step,
                double inv_bc2, OptTensor live) {
  const size_t count = p.size();
  if (count == 0) return;
  const bool eight = !ms.empty(), prox = !ref.empty();
  TORCH_CHECK(g.size() == count && m.size() == count && v.size() == count &&
                  keep.size() == count && ms.size() == vs.size() &&
                  (!eight || ms.size() == count) &&
                  (!prox || ref.size() == count),
              "adamw: the lists must have one entry a parameter");
  const torch::Device dev = p[0].device();
  TORCH_CHECK(dev.is_cuda(), "adamw: parameters must be on a GPU");
  const auto pt = p[0].scalar_type(), gt = g[0].scalar_type();
  auto real = [](torch::ScalarType t) {
    return t == torch::kFloat32 || t == torch::kBFloat16;
  };
  TORCH_CHECK(real(pt) && real(gt),
              "adamw: parameters and gradients must be float32 or bfloat16");
  const auto state = eight ? torch::kFloat8_e4m3fn : torch::kFloat32;
  std::vector<std::pair<uintptr_t, uintptr_t>> written, read;
  written.reserve(count * (eight ? 5 : 3));
  auto check = [&](const torch::Tensor& t, torch::ScalarType type, int64_t n,
                   bool out, const char* name) {
    TORCH_CHECK(t.device() == dev, "adamw: ", name, " is on ", t.device(),
                ", the first parameter on ", dev);
    TORCH_CHECK(t.scalar_type() == type, "adamw: ", name, " must be ", type,
                ", not ", t.scalar_type());
    TORCH_CHECK(t.is_contiguous() && t.numel() == n, "adamw: ", name,
                " must be contiguous with ", n, " elements");
    if (n > 0) {
      const auto a = reinterpret_cast<uintptr_t>(t.data_ptr());
      (out ? written : read).emplace_back(a, a + t.nbytes());
    }
  };
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = p[i].numel();
    check(p[i], pt, n, true, "a parameter");
    check(g[i], gt, n, false, "a gradient");
    check(m[i], state, n, true, "a first moment");
    check(v[i], state, n, true, "a second moment");
    if (eight) {
      const int64_t blocks = (n + kAdamwBlock - 1) / kAdamwBlock;
      check(ms[i], torch::kFloat32, blocks, true, "a first moment's scales");
      check(vs[i], torch::kFloat32, blocks, true, "a second moment's scales");
    }
    if (prox) check(ref[i], torch::kFloat32, n, false, "a reference");
    // as many elements in another order would be another tensor's step
    for (const auto* t : {&g[i], &m[i], &v[i], prox ? &ref[i] : &p[i]})
      TORCH_CHECK_VALUE(t->sizes() == p[i].sizes(), "adamw: ", t->sizes(),
                        " beside a parameter ", p[i].sizes());
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK(written[i - 1].second <= written[i].first,
                "adamw: a tensor that the step writes is there twice, or two "
                "of them overlap");
  for (const auto& [first, last] : read) {
    const auto next = std::lower_bound(
        written.begin(), written.end(), first,
        [](const auto& w, uintptr_t x) { return w.second <= x; });
    TORCH_CHECK(next == written.end() || last <= next->first,
                "adamw: a gradient or reference overlaps a tensor that the "
                "step writes");
  }
  AdamwScalars sc{};
  sc.b1 = static_cast<float>(b1);
  sc.omb1 = static_cast<float>(1.0 - b1);
  sc.b2 = static_cast<float>(b2);
  sc.omb2 = static_cast<float>(1.0 - b2);
  sc.eps = static_cast<float>(eps);
  sc.mu = static_cast<float>(mu);
  sc.step = static_cast<float>(step);
  sc.inv_bc2 = static_cast<float>(inv_bc2);
  if (live.has_value()) {
    check_gpu(*live, dev, "adamw: the live scalars");
    TORCH_CHECK(live->scalar_type() == torch::kFloat32 &&
                    live->is_contiguous() && live->numel() == 2,
                "adamw: the live scalars are two contiguous float32");
    for (const auto* ts : {&p, &m, &v, &ms, &vs})
      for (const auto& t : *ts)
        TORCH_CHECK(apart(*live, t), "adamw: the live scalars overlap a tensor "
                    "that the step writes");
    sc.live = live->data_ptr<float>();
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  AdamwTable tab{};
  int64_t grid = 0;
  auto flush = [&] {
    if (tab.count > 0) {
      launch_adamw(tab, sc, pt == torch::kBFloat16, gt == torch::kBFloat16,
                   eight, prox, stream());
      HIP_CHECK_LAST();
    }
    tab.count = 0;
    tab.aligned = 0;
    grid = 0;
  };
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = p[i].numel();
    if (n == 0) continue;
    const int64_t groups = (n + kAdamwChunk - 1) / kAdamwChunk;
    TORCH_CHECK(groups <= kMostBlocks, "adamw: a tensor of ", n,
                " elements is too long");
    if (tab.count == kAdamwTensors || grid + groups > kMostBlocks) flush();
    // whoever saved the parameter for a backward pass has to learn of this
    if (!p[i].is_inference()) p[i].unsafeGetTensorImpl()->bump_version();
    AdamwTensor& t = tab.t[tab.count];
    t.p = p[i].data_ptr();
    t.g = g[i].data_ptr();
    t.m = m[i].data_ptr();
    t.v = v[i].data_ptr();
    t.ms = eight ? ms[i].data_ptr<float>() : nullptr;
    t.vs = eight ? vs[i].data_ptr<float>() : nullptr;
    t.ref = prox ? ref[i].data_ptr<float>() : nullptr;
    t.n = n;
    // four elements at once: 16 bytes of fp32, 8 of bf16, 4 of codes
    auto at = [](const void* q, size_t unit) {
      return reinterpret_cast<uintptr_t>(q) % (4 * unit) == 0;
    };
    const size_t su = eight ? 1 : 4;
    if (at(t.p, p[i].element_size()) && at(t.g, g[i].element_size()) &&
        at(t.m, su) && at(t.v, su) && (!prox || at(t.ref, 4)))
      tab.aligned |= 1ull << tab.count;
    tab.keep[tab.count] = static_cast<float>(keep[i]);
    tab.first[tab.count] = static_cast<int>(grid);
    grid += groups;
    tab.first[++tab.count] = static_cast<int>(grid);
  }
  flush();
}

// ---- residual add + layer norm ----------------------------------------------
void check_norm(const torch::Tensor& x, const torch::Tensor& w,
                int64_t groups, int64_t* rows, int64_t* H) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.is_contiguous(),
              "add_norm: x must be a contiguous GPU tensor");
  *H = x.size(-1);
  TORCH_CHECK(*H >= 1 && *H <= kAddNormMaxH, "add_norm: rows of 1 to ",
              kAddNormMaxH, " elements, not ", *H);
  *rows = x.numel() / *H;
  TORCH_CHECK(groups >= 1 && groups <= 65535 && *rows % groups == 0,
              "add_norm: ", *rows, " rows do not divide into ", groups,
              " groups");
  const int64_t threads = *H <= 1024 ? 64 : *H <= 4096 ? 256 : 1024;  // a row
  TORCH_CHECK(*rows <= kMostThreads / threads - 3, "add_norm: too many rows (",
              *rows, ")");
  check_gpu(w, x.device(), "add_norm: weight");
  TORCH_CHECK(w.scalar_type() == torch::kFloat32 && w.is_contiguous() &&
                  w.numel() == groups * *H,
              "add_norm: weight and bias must be contiguous float32 with ",
              groups * *H, " elements");
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
add_norm_fwd(torch::Tensor x, OptTensor r, torch::Tensor w, torch::Tensor b,
             double eps, int64_t groups) {
  int64_t rows, H;
  const Elem type = elem_of(x, "add_norm: x");
  check_norm(x, w, groups, &rows, &H);
  check_norm(x, b, groups, &rows, &H);
  if (r.has_value()) {
    check_like(*r, x, "add_norm: residual");
    TORCH_CHECK(r->is_contiguous(), "add_norm: residual must be contiguous");
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto y = torch::empty_like(x);
  auto s = r.has_value() ? torch::empty_like(x) : x;
  const auto f32 = x.options().dtype(torch::kFloat32);
  auto mean = torch::empty({rows}, f32), inv = torch::empty({rows}, f32);
  if (rows == 0) return {y, s, mean, inv};
  AddNormFwd f{};
  f.x = x.data_ptr();
  f.r = r.has_value() ? r->data_ptr() : nullptr;
  f.w = w.data_ptr<float>();
  f.b = b.data_ptr<float>();
  f.s = s.data_ptr();
  f.y = y.data_ptr();
  f.mean = mean.data_ptr<float>();
  f.inv = inv.data_ptr<float>();
  f.rows = rows;
  f.groups = static_cast<int>(groups);
  f.H = static_cast<int>(H);
  f.eps = static_cast<float>(eps);
  const bool vec = H % 4 == 0 && aligned16(x) && aligned16(w) &&
                   aligned16(b) && (!r.has_value() || aligned16(*r));
  launch_add_norm_fwd(f, type, vec, stream());
  HIP_CHECK_LAST();
  return {y, s, mean, inv};
}

torch::Tensor add_norm_bwd(torch::Tensor gy, OptTensor gs, torch::Tensor s,
                           torch::Tensor w, torch::Tensor mean,
                           torch::Tensor inv, int64_t groups,
                           torch::Tensor dw, torch::Tensor db) {
  int64_t rows, H;
  const Elem type = elem_of(s, "add_norm: the sum");
  check_norm(s, w, groups, &rows, &H);
  check_norm(s, dw, groups, &rows, &H);
  check_norm(s, db, groups, &rows, &H);
  check_like(gy, s, "add_norm: the output's gradient");
  TORCH_CHECK(gy.is_contiguous(), "add_norm: gradients must be contiguous");
  if (gs.has_value()) {
    check_like(*gs, s, "add_norm: the sum's gradient");
    TORCH_CHECK(gs->is_contiguous(), "add_norm: gradients must be contiguous");
  }
  for (const auto& t : {mean, inv}) {
    check_gpu(t, s.device(), "add_norm: row statistics");
    TORCH_CHECK(t.scalar_type() == torch::kFloat32 && t.is_contiguous() &&
                    t.numel() == rows,
                "add_norm: row statistics must be ", rows, " float32");
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(s.device());
  auto gx = torch::empty_like(s);
  if (rows == 0) {
    dw.zero_();
    db.zero_();
    return gx;
  }
  const int parts =
      add_norm_parts(rows, static_cast<int>(groups), static_cast<int>(H));
  auto partials = torch::empty({groups, parts, 2, H},
                               s.options().dtype(torch::kFloat32));
  AddNormBwd b{};
  b.gy = gy.data_ptr();
  b.gs = gs.has_value() ? gs->data_ptr() : nullptr;
  b.s = s.data_ptr();
  b.w = w.data_ptr<float>();
  b.mean = mean.data_ptr<float>();
  b.inv = inv.data_ptr<float>();
  b.gx = gx.data_ptr();
  b.dw = dw.data_ptr<float>();
  b.db = db.data_ptr<float>();
  b.partials = partials.data_ptr<float>();
  b.rows = rows;
  b.groups = static_cast<int>(groups);
  b.H = static_cast<int>(H);
  b.parts = parts;
  const bool vec = H % 4 == 0 && aligned16(s) && aligned16(w) &&
                   aligned16(gy) && (!gs.has_value() || aligned16(*gs));
  launch_add_norm_bwd(b, type, vec, stream());
  HIP_CHECK_LAST();
  return gx;
}

// ---- masked attention ---------------------------------------------------------
// Elements from a token to the next.  A tile's 64 rows are addressed with 32
// bits of bytes: 63 x 2^25 x 2 and a row's 256 are less than 2^32.
constexpr int64_t kMostRow = 1 << 25;

// The kernels read 16 bytes at a time: rows of contiguous elements whose
// strides and start are multiples of 8 of them.  Anything else is copied
// (`contiguous` would return a contiguous tensor that starts off 16 bytes as it
// is).
torch::Tensor readable(const torch::Tensor& t) {
  bool ok = t.stride(3) == 1 && aligned16(t);
  for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0;
  // a copy's tokens are not further apart: `describe`
  ok = ok && t.stride(1) >= 0 && t.stride(1) <= kMostRow;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

HeadView view_of(const torch::Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

MaskedAttn describe(const torch::Tensor& q, const torch::Tensor& k,
                    const torch::Tensor& v, double scale, bool causal,
                    double softcap, const OptTensor& prefix,
                    const OptTensor& doc, const OptTensor& slopes) {
  TORCH_CHECK_TYPE(q.is_cuda() && (q.scalar_type() == torch::kBFloat16 ||
                                   q.scalar_type() == torch::kFloat16),
                   "attention: q must be a bfloat16 or float16 GPU tensor");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() &&
                        q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                        q.size(3) == k.size(3),
                    "attention takes q [N, S, H, D] and k, v [N, S, Hkv, D], "
                    "got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  auto here = [&](const torch::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.device() == q.device(), "attention: ", name, " on ",
                      t.device(), ", q on ", q.device());
  };
  for (const auto& t : {k, v}) {
    TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(),
                     "attention: q, k and v must have one type, got ",
                     q.scalar_type(), ", ", k.scalar_type(), ", ",
                     v.scalar_type());
    here(t, "k or v");
  }
  const int64_t N = q.size(0), S = q.size(1), H = q.size(2), Hkv = k.size(2),
                D = q.size(3);
  TORCH_CHECK_VALUE(Hkv >= 1 && H % Hkv == 0, "attention: ", H,
                    " heads do not divide over ", Hkv, " key heads");
  TORCH_CHECK_VALUE(D >= 8 && D <= 128 && D % 8 == 0,
                    "attention: head sizes are multiples of 8 up to 128, not ",
                    D);
  constexpr int64_t kMost = std::numeric_limits<int>::max();
  TORCH_CHECK_VALUE(
      S <= (1 << 22) && N <= kMost && H <= kMost && N * H <= kMost &&
          N * H * ((S + 63) / 64) <= kMostBlocks,
      "attention: too many tokens (a sequence has at most 2^22, all heads of "
      "all sequences 2^24 tiles of 64)");
  TORCH_CHECK_VALUE(H * D <= kMostRow, "attention: all heads of a token have "
                    "at most ", kMostRow, " elements, not ", H * D);
  // the kernels form scale / softcap and slope / scale in fp32
  TORCH_CHECK_VALUE(scale >= 1e-18 && scale <= 1e18,
                    "attention: the scale must be within 1e-18 and 1e18, got ",
                    scale);
  TORCH_CHECK_VALUE(
      softcap == 0.0 || (softcap >= 1e-18 && softcap <= 1e18),
      "attention: softcap must be 0 or within 1e-18 and 1e18, got ", softcap);
  MaskedAttn a{};
  a.N = static_cast<int>(N);
  a.S = static_cast<int>(S);
  a.H = static_cast<int>(H);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.causal = causal;
  a.scale = static_cast<float>(scale);
  a.softcap = static_cast<float>(softcap);
  if (prefix.has_value()) {
    TORCH_CHECK_VALUE(causal,
                      "attention: a prefix widens a causal mask: causal=True");
    here(*prefix, "prefix");
    TORCH_CHECK_VALUE(prefix->scalar_type() == torch::kInt32 &&
                          prefix->dim() == 1 && prefix->size(0) == N &&
                          prefix->is_contiguous(),
                      "attention: prefix must be int32 [", N, "]");
    a.prefix = prefix->data_ptr<int>();
  }
  if (doc.has_value()) {
    here(*doc, "doc");
    TORCH_CHECK_VALUE(doc->scalar_type() == torch::kInt32 &&
                          doc->dim() == 2 && doc->size(0) == N &&
                          doc->size(1) == S && doc->is_contiguous(),
                      "attention: doc must be int32 [", N, ", ", S, "]");
    a.doc = doc->data_ptr<int>();
  }
  if (slopes.has_value()) {
    here(*slopes, "slopes");
    TORCH_CHECK_VALUE(slopes->scalar_type() == torch::kFloat32 &&
                          slopes->dim() == 1 && slopes->size(0) == H &&
                          slopes->is_contiguous(),
                      "attention: slopes must be float32 [", H, "]");
    a.slopes = slopes->data_ptr<float>();
  }
  return a;
}

// (o [N, S, H, D], what rounding took from it: empty if no backward pass
// follows; row statistics, summary of doc: empty if there is none)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
masked_attn_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                double scale, bool causal, double softcap, OptTensor prefix,
                OptTensor doc, OptTensor slopes, bool train) {
  MaskedAttn a =
      describe(q, k, v, scale, causal, softcap, prefix, doc, slopes);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto o = torch::empty({a.N, a.S, a.H, a.D}, q.options());
  auto rest = torch::empty({train ? o.numel() : 0}, q.options());
  auto lse = torch::empty({a.N, a.H, a.S}, q.options().dtype(torch::kFloat32));
  const int64_t tiles = (a.S + kAttnGroup - 1) / kAttnGroup;
  const bool summary = doc.has_value() && a.S > kAttnShort;
  auto sum = torch::empty({summary ? a.N * tiles : 0, 4},
                          q.options().dtype(torch::kInt32));
  if (o.numel() == 0) return {o, rest, lse, sum};
  q = readable(q);
  k = readable(k);
  v = readable(v);
  a.q = view_of(q);
  a.k = view_of(k);
  a.v = view_of(v);
  a.o = view_of(o);
  a.lse = lse.data_ptr<float>();
  if (train) a.rest = rest.data_ptr();
  if (summary) {
    a.tiles = reinterpret_cast<int4*>(sum.data_ptr<int>());
    launch_masked_attn_tiles(a, stream());
  }
  launch_masked_attn_fwd(a, elem_of(q, "q"), stream());
  HIP_CHECK_LAST();
  return {o, rest, lse, sum};
}

// Writes gq, gk, gv: any layout whose rows are contiguous and whose strides
// and start are multiples of 8 elements.
void masked_attn_bwd(torch::Tensor go, torch::Tensor q, torch::Tensor k,
                     torch::Tensor v, torch::Tensor o, torch::Tensor rest,
                     torch::Tensor lse, torch::Tensor sum, torch::Tensor gq,
                     torch::Tensor gk, torch::Tensor gv, double scale,
                     bool causal, double softcap, OptTensor prefix,
                     OptTensor doc, OptTensor slopes) {
  MaskedAttn a =
      describe(q, k, v, scale, causal, softcap, prefix, doc, slopes);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  check_like(go, q, "masked_attn: the output's gradient");
  check_like(o, q, "masked_attn: the output");
  check_gpu(rest, q.device(), "masked_attn: the output's rest");
  TORCH_CHECK(rest.scalar_type() == q.scalar_type() && rest.is_contiguous() &&
                  rest.numel() == q.numel() && aligned16(rest),
              "masked_attn: the output's rest does not match");
  check_like(gq, q, "masked_attn: q's gradient");
  check_like(gk, k, "masked_attn: k's gradient");
  check_like(gv, v, "masked_attn: v's gradient");
  check_gpu(lse, q.device(), "masked_attn: row statistics");
  check_gpu(sum, q.device(), "masked_attn: summary");
  const int64_t tiles = (a.S + kAttnGroup - 1) / kAttnGroup;
  const int64_t entries =
      doc.has_value() && a.S > kAttnShort ? a.N * tiles * 4 : 0;
  TORCH_CHECK(lse.scalar_type() == torch::kFloat32 && lse.is_contiguous() &&
                  lse.numel() == static_cast<int64_t>(a.N) * a.H * a.S,
              "masked_attn: row statistics do not match");
  TORCH_CHECK(sum.scalar_type() == torch::kInt32 && sum.is_contiguous() &&
                  sum.numel() == entries,
              "masked_attn: the summary does not match");
  for (const auto& t : {gq, gk, gv}) {
    bool ok = t.stride(3) == 1 && aligned16(t);
    for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0;
    TORCH_CHECK(ok, "masked_attn: gradients need contiguous rows at 16 bytes");
  }
  if (q.numel() == 0) {
    gk.zero_();
    gv.zero_();
    return;
  }
  q = readable(q);
  k = readable(k);
  v = readable(v);
  go = readable(go);
  o = readable(o);
  auto delta = torch::empty_like(lse);
  a.q = view_of(q);
  a.k = view_of(k);
  a.v = view_of(v);
  a.o = view_of(o);
  a.go = view_of(go);
  a.gq = view_of(gq);
  a.gk = view_of(gk);
  a.gv = view_of(gv);
  a.rest = rest.data_ptr();
  a.lse = lse.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  if (sum.numel() > 0) a.tiles = reinterpret_cast<int4*>(sum.data_ptr<int>());
  a.shares = masked_attn_shares(a);
  torch::Tensor partial;
  if (a.shares > 1) {
    partial = torch::empty({2, a.shares, a.N, a.S, a.Hkv, a.D},
                           lse.options());
    a.partial = partial.data_ptr<float>();
  }
  launch_masked_attn_bwd(a, elem_of(q, "q"), stream());
  HIP_CHECK_LAST();
}

// ---- autograd -------------------------------------------------------------------
// In C++: the engine's thread then needs no interpreter, which is most of a
// small backward pass (norm of 4096 x 768, forward and backward: 115 us of
// host time with functions in Python, 86 here).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The kernels' gradients have no gradient of their own: asked for one
// (create_graph), they raise when it is used, as once_differentiable's do.
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list there;
  for (auto& g : grads)
    if (g.defined()) there.push_back(g.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice ") + name +
          ", whose backward pass is a kernel",
      static_cast<int64_t>(there.size()));
  auto marked = (*error)(std::move(there));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

struct AddNormFn : public torch::autograd::Function<AddNormFn> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor x,
                               OptTensor residual, torch::Tensor weight,
                               torch::Tensor bias, double eps, int64_t groups,
                               OptTensor gslot_w, OptTensor gslot_b) {
    auto [y, s, mean, inv] =
        add_norm_fwd(x, residual, weight, bias, eps, groups);
    ctx->save_for_backward({s, weight, mean, inv});
    // Not saved as operands: they are written here, and they are views of a
    // buffer that every other gradient is added into meanwhile.
    if (gslot_w.has_value()) {
      ctx->saved_data["gslot_w"] = *gslot_w;
      ctx->saved_data["gslot_b"] = *gslot_b;
    }
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["bias"] = bias.sizes().vec();
    ctx->set_materialize_grads(false);
    if (!residual.has_value()) s = s.view_as(s);  // no output is an input
    return {y, s};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool residual = ctx->saved_data["residual"].toBool();
    variable_list out(8);
    torch::Tensor gx;
    if (!grads[0].defined()) {  // only the sum was used
      gx = grads[1];
      if (ctx->saved_data.count("gslot_w") > 0) {
        ctx->saved_data["gslot_w"].toTensor().zero_();
        ctx->saved_data["gslot_b"].toTensor().zero_();
      }
    } else {
      const auto& weight = saved[1];
      const bool direct = ctx->saved_data.count("gslot_w") > 0;
      auto gw = direct ? ctx->saved_data["gslot_w"].toTensor()
                       : torch::empty_like(weight);
      auto gb = direct ? ctx->saved_data["gslot_b"].toTensor()
                       : torch::empty(ctx->saved_data["bias"].toIntVector(),
                                      weight.options());
      OptTensor gs;
      if (grads[1].defined()) gs = grads[1].contiguous();
      gx = add_norm_bwd(grads[0].contiguous(), gs, saved[0], weight, saved[2],
                        saved[3], ctx->saved_data["groups"].toInt(), gw, gb);
      if (!direct) {
        out[2] = gw;
        out[3] = gb;
      }
    }
    out[0] = gx;
    if (residual && ctx->needs_input_grad(1)) out[1] = gx;
    return once("add + layer norm", std::move(out));
  }
};

std::tuple<torch::Tensor, torch::Tensor> add_layer_norm(
    torch::Tensor x, OptTensor residual, torch::Tensor weight,
    torch::Tensor bias, double eps, int64_t groups, OptTensor gslot_w,
    OptTensor gslot_b) {
  for (const auto& g : {gslot_w, gslot_b}) {
    if (!g.has_value()) continue;
    check_gpu(*g, x.device(), "add_norm: a gradient slot");
    TORCH_CHECK(g->scalar_type() == torch::kFloat32 && g->is_contiguous() &&
                    g->numel() == weight.numel(),
                "add_norm: gradient slots must be contiguous float32 of "
                "weight's size");
    // one launch writes both, column by column
    TORCH_CHECK(apart(*g, weight) && apart(*g, bias),
                "add_norm: gradient slots must not overlap the parameters");
  }
  TORCH_CHECK(!gslot_w.has_value() || !gslot_b.has_value() ||
                  apart(*gslot_w, *gslot_b),
              "add_norm: gradient slots must not overlap each other");
  auto out = AddNormFn::apply(x, residual, weight, bias, eps, groups, gslot_w,
                              gslot_b);
  return {out[0], out[1]};
}

void keep_masks(AutogradContext* ctx, double scale, bool causal,
                double softcap, variable_list saved, const OptTensor& prefix,
                const OptTensor& doc, const OptTensor& slopes) {
  for (const auto& t : {prefix, doc, slopes})
    saved.push_back(t.value_or(torch::Tensor()));
  ctx->save_for_backward(std::move(saved));
  ctx->saved_data["scale"] = scale;
  ctx->saved_data["causal"] = causal;
  ctx->saved_data["softcap"] = softcap;
}

void run_masked_bwd(AutogradContext* ctx, const torch::Tensor& go,
                    const torch::Tensor& q, const torch::Tensor& k,
                    const torch::Tensor& v, const variable_list& saved,
                    size_t at, torch::Tensor gq, torch::Tensor gk,
                    torch::Tensor gv) {
  auto opt = [&](size_t i) -> OptTensor {
    return saved[i].defined() ? OptTensor(saved[i]) : OptTensor();
  };
  masked_attn_bwd(go, q, k, v, saved[at], saved[at + 1], saved[at + 2],
                  saved[at + 3], gq, gk, gv,
                  ctx->saved_data["scale"].toDouble(),
                  ctx->saved_data["causal"].toBool(),
                  ctx->saved_data["softcap"].toDouble(), opt(at + 4),
                  opt(at + 5), opt(at + 6));
}

struct MaskedAttnFn : public torch::autograd::Function<MaskedAttnFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor q,
                               torch::Tensor k, torch::Tensor v, double scale,
                               bool causal, double softcap, OptTensor prefix,
                               OptTensor doc, OptTensor slopes, bool train) {
    auto [o, rest, lse, sum] = masked_attn_fwd(
        q, k, v, scale, causal, softcap, prefix, doc, slopes, train);
    keep_masks(ctx, scale, causal, softcap, {q, k, v, o, rest, lse, sum},
               prefix, doc, slopes);
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(10);
    for (int i = 0; i < 3; ++i)
      out[i] = torch::empty(saved[i].sizes(), saved[i].options());
    run_masked_bwd(ctx, grads[0], saved[0], saved[1], saved[2], saved, 3,
                   out[0], out[1], out[2]);
    return once("masked attention", std::move(out));
  }
};

// The fused projection's layout [N, S, 3, H, D]: one gradient tensor, written
// in place of three that autograd would have to put together.
struct MaskedAttnQKVFn : public torch::autograd::Function<MaskedAttnQKVFn> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor qkv,
                               double scale, bool causal, double softcap,
                               OptTensor prefix, OptTensor doc,
                               OptTensor slopes, bool train) {
    auto [o, rest, lse, sum] = masked_attn_fwd(
        qkv.select(2, 0), qkv.select(2, 1), qkv.select(2, 2), scale, causal,
        softcap, prefix, doc, slopes, train);
    keep_masks(ctx, scale, causal, softcap, {qkv, o, rest, lse, sum}, prefix,
               doc, slopes);
    return o;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto& qkv = saved[0];
    variable_list out(8);
    auto g = torch::empty(qkv.sizes(), qkv.options());
    run_masked_bwd(ctx, grads[0], qkv.select(2, 0), qkv.select(2, 1),
                   qkv.select(2, 2), saved, 1, g.select(2, 0), g.select(2, 1),
                   g.select(2, 2));
    out[0] = g;
    return once("masked attention", std::move(out));
  }
};

// masks as the kernels read them
struct Masks {
  OptTensor prefix, doc, slopes;

  Masks(const OptTensor& p, const OptTensor& d, const OptTensor& s) {
    if (p.has_value()) prefix = p->contiguous();
    if (d.has_value()) doc = d->contiguous();
    if (s.has_value()) {
      TORCH_CHECK_VALUE(!s->requires_grad(),
                        "attention: slopes are constants: they get no "
                        "gradient");
      slopes = s->contiguous();
    }
  }
};

torch::Tensor masked_attention(torch::Tensor q, torch::Tensor k,
                               torch::Tensor v, double scale, bool causal,
                               double softcap, OptTensor prefix, OptTensor doc,
                               OptTensor slopes) {
  const Masks m(prefix, doc, slopes);
  const bool train = at::GradMode::is_enabled() &&
                     (q.requires_grad() || k.requires_grad() ||
                      v.requires_grad());
  return MaskedAttnFn::apply(q, k, v, scale, causal, softcap, m.prefix, m.doc,
                             m.slopes, train);
}

// [N, S, H * D]
torch::Tensor masked_attention_qkv(torch::Tensor qkv, double scale,
                                   bool causal, double softcap,
                                   OptTensor prefix, OptTensor doc,
                                   OptTensor slopes) {
  const Masks m(prefix, doc, slopes);
  const bool train = at::GradMode::is_enabled() && qkv.requires_grad();
  return MaskedAttnQKVFn::apply(qkv, scale, causal, softcap, m.prefix, m.doc,
                                m.slopes, train)
      .flatten(2);
}

}  // namespace

void bind_encoder(pybind11::module& m) {
  m.def("adamw_step", &adamw_step);
  m.def("add_layer_norm", &add_layer_norm);
  m.def("masked_attention", &masked_attention);
  m.def("masked_attention_qkv", &masked_attention_qkv);
}

}  // namespace colearn
