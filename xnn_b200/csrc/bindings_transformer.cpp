// Python bindings and autograd nodes of the transformer operators (attention.cu, dropout.cu, embedding.cu),
// launched on the current stream of the operands' device; workspaces come from the caching allocator on that stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <array>
#include <cmath>
#include <limits>

#include "attention.h"
#include "attention_params.h"

template <typename T>
cudaError_t counter_dropout(int64_t outer, int64_t shared, int64_t inner, double p, const int64_t* rng, const T* x, T* y,
                            cudaStream_t s);
template <typename T, typename I>
cudaError_t embedding_lookup(int64_t N, int64_t V, int C, const T* table, const I* ids, double scale, T* out, cudaStream_t s);
template <typename T, typename I>
cudaError_t embedding_grad(int64_t N, int64_t V, int C, const I* ids, const T* g, double scale, int* ints, T* partials,
                           T* table, cudaStream_t s);
int64_t embedding_grad_ints(int64_t N, int64_t V, int64_t C);
int64_t embedding_grad_partials(int64_t N, int64_t V, int64_t C);

namespace {

#define XNN_OK(call)                                                                          \
  do {                                                                                        \
    const cudaError_t err_ = (call);                                                          \
    TORCH_CHECK(err_ == cudaSuccess, #call, " failed: ", cudaGetErrorString(err_));           \
  } while (0)

// The kernels carry no tangents: a call or a backward pass over a dual tensor would drop them without a word.
void no_tangents(const char* what, std::initializer_list<torch::Tensor> tensors) {
  for (const auto& t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " on CUDA has no forward-mode derivative");
}

// A trace records operators that PyTorch knows; a result of these kernels would become a constant in it.
void not_traced(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " on CUDA cannot be traced (torch.jit.trace)");
}

constexpr int ANY_LENGTH = std::numeric_limits<int>::max();
constexpr int SHORT = 32;            // rows of the square tiles that hold a short structure whole
constexpr int SMS = 148;

void check_rows(const torch::Tensor& t, const torch::Tensor& like, int64_t N, int64_t heads, int64_t D, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type(), "structure attention: ",
              name, " must be on ", like.device(), " with the dtype of q");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == N && t.size(1) == heads && t.size(2) == D && (D == 1 || N == 0 || t.stride(2) == 1),
              "structure attention: ", name, " must be (", N, ", ", heads, ", ", D, ") with contiguous rows");
}

// the parameters that every pass shares; strides of a size-one dimension do not matter
template <typename T>
attn::Params<T> make_params(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ptr,
                            const c10::optional<torch::Tensor>& mask, double scale) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, "structure attention: q (atoms, heads, width) on a CUDA device");
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2), HK = k.dim() == 3 ? k.size(1) : 0;
  TORCH_CHECK(HK > 0 && H > 0 && H % HK == 0 && H <= 65535, "structure attention: ", H, " heads over ", HK, " key heads");
  TORCH_CHECK(D > 0 && D <= 128 && N < (1 << 30), "structure attention: width 1 .. 128, fewer than 2^30 atoms");
  check_rows(q, q, N, H, D, "q");
  check_rows(k, q, N, HK, D, "k");
  check_rows(v, q, N, HK, D, "v");
  TORCH_CHECK(ptr.device() == q.device() && ptr.scalar_type() == torch::kInt64 && ptr.dim() == 1 && ptr.is_contiguous() &&
                  ptr.numel() >= 1 && ptr.numel() < (1 << 30), "structure attention: ptr must be int64 (structures + 1) on ", q.device());
  TORCH_CHECK((N / SHORT + ptr.numel() + 2) * 3 * H < std::numeric_limits<int>::max(),
              "structure attention: more structures and heads than a launch can number");
  attn::Params<T> p{};
  p.q = q.data_ptr<T>(); p.qs = q.stride(0); p.qh = q.stride(1);
  p.k = k.data_ptr<T>(); p.ks = k.stride(0); p.kh = k.stride(1);
  p.v = v.data_ptr<T>(); p.vs = v.stride(0); p.vh = v.stride(1);
  p.ptr = ptr.data_ptr<int64_t>();
  if (mask.has_value()) {
    TORCH_CHECK(mask->device() == q.device() && mask->scalar_type() == torch::kBool && mask->dim() == 1 &&
                    mask->size(0) == N && mask->is_contiguous(), "structure attention: key_mask must be bool (atoms) on ", q.device());
    p.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr<bool>());
  }
  p.scale = (T)scale;
  p.N = (int)N; p.num = (int)ptr.numel() - 1; p.H = (int)H; p.HK = (int)HK; p.D = (int)D;
  p.splits = 1;
  p.max_len = ANY_LENGTH;
  p.rest = 1;
  return p;
}

// Which kernels take a call. Structures of at most SHORT atoms fill a square tile of the FP32 / FP64 pipes; the tensor cores
// own 128 rows at a time (float64: 32), most of them empty for such a structure.
//   all within SHORT                       the short kernels
//   one wave of structures and heads, or
//   LONG_AVERAGE atoms on average          the tensor cores for all
//   otherwise                              the tensor cores for the structures above SHORT, the short kernels for the rest
// Both ways, for all / in two launches, forward, backward, second derivative at 64 columns in us: 64 structures of 9-40 atoms,
// one head 11, 17, 39 / 16, 27, 55; of 400 x 2 heads 37, 138, 259 / 35, 77, 172; of 20-60 atoms 41, 149, 306 / 47, 135, 278.
// float64: 11, 29, 73 / 20, 44, 105; 74, 183, 371 / 66, 142, 343; 103, 263, 618 / 108, 253, 615. float32 of more than 64
// columns, whose long second derivatives are attention_f64.cu's, one after the other forward, backward and that: 64 structures
// of 20-50 atoms x 1 x 128 154 / 190, of 9-40 150 / 183, 64 of 30-60 x 4 x 128 533 / 597, 300 of 30-60 x 1 x 72 465 / 529.
constexpr int LONG_AVERAGE = 40, TC_SECOND_WIDTH = 64, TC_ROWS = 128, TC_TILE = 64;

struct Plan { bool long_ones, short_ones; };

template <typename T>
Plan choose(const attn::Params<T>& p, int64_t max_len) {
  if (max_len <= SHORT) return {false, true};
  return {true, (int64_t)p.N < LONG_AVERAGE * (int64_t)p.num && (int64_t)p.num * p.H > SMS};
}

// The parameters of the two launches: the long structures, the short ones (with the rows of none, where both run). The
// tensor cores' blocks and workspace are then numbered without regard to the short ones, of which there may be many.
template <typename T>
attn::Params<T> long_part(attn::Params<T> p, const Plan& plan) {
  if (plan.short_ones) {
    p.min_len = SHORT + 1;
    p.rest = 0;
    p.compact = sizeof(T) == 4;
  }
  return p;
}
template <typename T>
attn::Params<T> short_part(attn::Params<T> p, const Plan& plan) {
  if (plan.long_ones) p.max_len = SHORT;
  return p;
}

// How many blocks share the walk over the other axis (their partial results are added in order). With `slots` blocks running
// at a time, z shares take ceil(blocks z / slots) rounds of walk / z tiles and a fixed part of about two tiles (staging,
// storing); up to 16 shares, of two tiles at least, and only for a tenth less time, as the sums are another pass.
int choose_splits(int64_t row_blocks, int64_t max_len, int tile, int slots) {
  const int64_t walk = (max_len + tile - 1) / tile;
  int best = 1;
  double least = 0;
  for (int z = 1; z <= 16 && (z == 1 || walk >= 2 * z); ++z) {
    const double cost = (double)((row_blocks * z + slots - 1) / slots) * (double)((walk + z - 1) / z + 2);
    if (z == 1 || cost < 0.9 * least) {
      best = z;
      least = cost;
    }
  }
  return best;
}
template <typename T>
int splits_of(const attn::Params<T>& p, int heads, int64_t max_len, bool tc = sizeof(T) == 4, int resident = 1) {
  const int rows = tc ? TC_ROWS : SHORT;
  const int64_t structures = p.min_len > 0 ? std::min(p.num, p.N / p.min_len) : p.num;
  const int64_t blocks = ((int64_t)p.N / rows + std::max<int64_t>(structures, 1)) * heads;
  return choose_splits(blocks, std::min<int64_t>(max_len, p.N), TC_TILE, SMS * resident);
}

torch::Tensor bytes(int64_t n, const torch::Tensor& like) { return torch::empty({n}, like.options().dtype(torch::kUInt8)); }

int* status_of(const torch::Tensor& status, const torch::Tensor& q) {
  TORCH_CHECK(status.device() == q.device() && status.scalar_type() == torch::kInt32 && status.numel() >= 1,
              "structure attention: an int32 status word on ", q.device());
  return status.data_ptr<int>();
}

template <typename T>
std::vector<torch::Tensor> forward_typed(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                         const torch::Tensor& ptr, const c10::optional<torch::Tensor>& mask, int64_t max_len,
                                         double scale, bool want_stats, const torch::Tensor& status) {
  auto p = make_params<T>(q, k, v, ptr, mask, scale);
  torch::Tensor out = torch::empty({p.N, p.H, p.D}, q.options());
  torch::Tensor lse;
  if (want_stats) lse = torch::empty({p.H, p.N}, q.options());
  if (p.N == 0) return {out, want_stats ? lse : out};
  const auto s = at::cuda::getCurrentCUDAStream();
  p.out0 = out.data_ptr<T>();
  p.lse = want_stats ? lse.data_ptr<T>() : nullptr;
  const auto plan = choose(p, max_len);
  if (plan.long_ones) {
    auto pl = long_part(p, plan);
    pl.splits = splits_of(pl, p.H, max_len, sizeof(T) == 4, p.D <= 64 ? 2 : 1);
    torch::Tensor work, images;
    if (pl.splits > 1) {
      work = torch::empty({(int64_t)pl.splits * p.H * p.N * (p.D + 2)}, q.options());
      pl.work = work.data_ptr<T>();
    }
    if constexpr (sizeof(T) == 4) {
      images = bytes(attn::tc_forward_bytes(pl), q);
      XNN_OK(attn::tc_forward(pl, static_cast<char*>(images.data_ptr()), status_of(status, q), s));
    } else {
      XNN_OK(attn::forward64(pl, s));
    }
    if (pl.splits > 1) XNN_OK(attn::forward_join<T>(pl, s));             // short structures' rows hold nothing yet
  }
  if (plan.short_ones) XNN_OK(attn::forward<T>(short_part(p, plan), s));
  return {out, want_stats ? lse : out};
}

template <typename T>
void set_outputs(attn::Params<T>& p, const torch::Tensor& go, const torch::Tensor& o, const torch::Tensor& lse,
                 const torch::Tensor& q) {
  check_rows(go, q, p.N, p.H, p.D, "the output's gradient");
  check_rows(o, q, p.N, p.H, p.D, "the output");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == q.scalar_type() && lse.is_contiguous() &&
                  lse.numel() == (int64_t)p.H * p.N, "structure attention: row statistics of another call");
  p.go = go.data_ptr<T>(); p.gos = go.stride(0); p.goh = go.stride(1);
  p.o = o.data_ptr<T>(); p.os = o.stride(0); p.oh = o.stride(1);
  p.lse = lse.data_ptr<T>();
}

template <typename T>
std::vector<torch::Tensor> backward_typed(const torch::Tensor& go, const torch::Tensor& q, const torch::Tensor& k,
                                          const torch::Tensor& v, const torch::Tensor& o, const torch::Tensor& lse,
                                          const torch::Tensor& ptr, const c10::optional<torch::Tensor>& mask, int64_t max_len,
                                          double scale, const torch::Tensor& status) {
  auto p = make_params<T>(q, k, v, ptr, mask, scale);
  set_outputs(p, go, o, lse, q);
  torch::Tensor dq = torch::empty({p.N, p.H, p.D}, q.options()), dk = torch::empty({p.N, p.HK, p.D}, q.options()),
       dv = torch::empty({p.N, p.HK, p.D}, q.options());
  if (p.N == 0) return {dq, dk, dv};
  const auto s = at::cuda::getCurrentCUDAStream();
  p.out0 = dq.data_ptr<T>(); p.out1 = dk.data_ptr<T>(); p.out2 = dv.data_ptr<T>();
  const auto plan = choose(p, max_len);
  if (plan.long_ones) {
    auto pl = long_part(p, plan);
    const int64_t nq = (int64_t)p.N * p.H * p.D, nk = (int64_t)p.N * p.HK * p.D;
    const int sq = splits_of(pl, p.H, max_len), sk = splits_of(pl, p.HK, max_len);
    torch::Tensor work, scratch;
    if (sq > 1 || sk > 1) {
      work = torch::empty({(sq > 1 ? sq * nq : 0) + (sk > 1 ? 2 * sk * nk : 0)}, q.options());
      pl.work = work.data_ptr<T>();
      pl.work_k = pl.work + (sq > 1 ? sq * nq : 0);
    }
    pl.splits = sq;
    pl.splits_k = sk;
    if constexpr (sizeof(T) == 4) {
      scratch = bytes(attn::tc_backward_bytes(pl), q);
      XNN_OK(attn::tc_backward(pl, static_cast<char*>(scratch.data_ptr()), status_of(status, q), s));
    } else {
      scratch = torch::empty({p.H, p.N}, q.options());
      pl.delta = scratch.data_ptr<T>();
      XNN_OK(attn::backward64(pl, s));
    }
    if (sq > 1) XNN_OK(attn::sum_splits<T>(nq, sq, pl.work, p.out0, nullptr, s));
    if (sk > 1) XNN_OK(attn::sum_splits<T>(nk, sk, pl.work_k, p.out1, p.out2, s));
  }
  if (plan.short_ones) XNN_OK(attn::backward_short<T>(short_part(p, plan), s));
  return {dq, dk, dv};
}

template <typename T>
std::vector<torch::Tensor> second_typed(const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& c,
                                        const torch::Tensor& go, const torch::Tensor& q, const torch::Tensor& k,
                                        const torch::Tensor& v, const torch::Tensor& o, const torch::Tensor& lse,
                                        const torch::Tensor& ptr, const c10::optional<torch::Tensor>& mask, int64_t max_len, double scale,
                                        const torch::Tensor& status) {
  auto p = make_params<T>(q, k, v, ptr, mask, scale);
  set_outputs(p, go, o, lse, q);
  check_rows(a, q, p.N, p.H, p.D, "the cotangent of dq");
  check_rows(b, q, p.N, p.HK, p.D, "the cotangent of dk");
  check_rows(c, q, p.N, p.HK, p.D, "the cotangent of dv");
  p.ca = a.data_ptr<T>(); p.cas = a.stride(0); p.cah = a.stride(1);
  p.cb = b.data_ptr<T>(); p.cbs = b.stride(0); p.cbh = b.stride(1);
  p.cc = c.data_ptr<T>(); p.ccs = c.stride(0); p.cch = c.stride(1);
  torch::Tensor q2 = torch::empty({p.N, p.H, p.D}, q.options()), k2 = torch::empty({p.N, p.HK, p.D}, q.options()),
       v2 = torch::empty({p.N, p.HK, p.D}, q.options()), do2 = torch::empty({p.N, p.H, p.D}, q.options());
  if (p.N == 0) return {q2, k2, v2, do2};
  const auto s = at::cuda::getCurrentCUDAStream();
  p.out0 = q2.data_ptr<T>(); p.out1 = k2.data_ptr<T>(); p.out2 = v2.data_ptr<T>(); p.out3 = do2.data_ptr<T>();
  const auto plan = choose(p, max_len);
  if (plan.long_ones) {
    const bool tc = sizeof(T) == 4 && p.D <= TC_SECOND_WIDTH;
    auto pl = long_part(p, plan);
    if (!tc) pl.compact = 0;
    const int sq = splits_of(pl, p.H, max_len, tc), sk = splits_of(pl, p.HK, max_len, tc);
    const int64_t nq = (int64_t)p.N * p.H * p.D, nk = (int64_t)p.N * p.HK * p.D;
    pl.splits = sq;
    pl.splits_k = sk;
    if constexpr (sizeof(T) == 4) {
      if (tc) {
        torch::Tensor work;
        if (sq > 1 || sk > 1) {
          work = torch::empty({(sq > 1 ? sq * nq : 0) + (sk > 1 ? 2 * sk * nk : 0)}, q.options());
          pl.work = work.data_ptr<T>();
          pl.work_k = pl.work + (sq > 1 ? sq * nq : 0);
        }
        auto images = bytes(attn::tc_second_bytes(pl), q);
        XNN_OK(attn::tc_second(pl, static_cast<char*>(images.data_ptr()), status_of(status, q), s));
        if (sq > 1) XNN_OK(attn::sum_splits<T>(nq, sq, pl.work, p.out0, nullptr, s));
        if (sk > 1) XNN_OK(attn::sum_splits<T>(nk, sk, pl.work_k, p.out1, p.out2, s));
      }
    }
    if (!tc) {
      torch::Tensor work = torch::empty({attn::second64_words<T>(pl)}, q.options().dtype(torch::kFloat64));
      XNN_OK(attn::second64<T>(pl, work.data_ptr<double>(), s));
    }
  }
  if (plan.short_ones) XNN_OK(attn::second_short<T>(short_part(p, plan), s));
  return {q2, k2, v2, do2};
}

using Tensors = std::vector<torch::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

Tensors attention_forward(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ptr,
                          const c10::optional<torch::Tensor>& mask, int64_t max_len, double scale, bool want_stats, const torch::Tensor& status) {
  const c10::cuda::CUDAGuard guard(q.device());
  Tensors r;
  AT_DISPATCH_FLOATING_TYPES(q.scalar_type(), "structure attention",
                             [&] { r = forward_typed<scalar_t>(q, k, v, ptr, mask, max_len, scale, want_stats, status); });
  return r;
}

Tensors attention_backward(const torch::Tensor& go, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                           const torch::Tensor& o, const torch::Tensor& lse, const torch::Tensor& ptr,
                           const c10::optional<torch::Tensor>& mask, int64_t max_len, double scale, const torch::Tensor& status) {
  const c10::cuda::CUDAGuard guard(q.device());
  Tensors r;
  AT_DISPATCH_FLOATING_TYPES(q.scalar_type(), "structure attention backward",
                             [&] { r = backward_typed<scalar_t>(go, q, k, v, o, lse, ptr, mask, max_len, scale, status); });
  return r;
}

torch::Tensor rows(const torch::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

c10::optional<torch::Tensor> maybe(const torch::Tensor& t) {
  return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt;
}

// The autograd nodes are C++: a backward pass runs on the engine's thread without the interpreter, which
// for the smallest calls costs more than the kernels. What the passes share beyond the saved tensors:
struct Setting { int64_t max_len; double scale; };
void keep(AutogradContext* ctx, const Setting& s) {
  ctx->saved_data["max_len"] = s.max_len;
  ctx->saved_data["scale"] = s.scale;
}
Setting kept(AutogradContext* ctx) { return {ctx->saved_data["max_len"].toInt(), ctx->saved_data["scale"].toDouble()}; }

// the gradients of <a, dq> + <b, dk> + <c, dv> in do, q, k, v; a node of its own, so that a third derivative
// meets it on every path to the inputs and is refused
struct AttentionSecond : torch::autograd::Function<AttentionSecond> {
  static variable_list forward(AutogradContext*, Variable a, Variable b, Variable c, Variable go, Variable q, Variable k,
                               Variable v, Variable o, Variable lse, Variable ptr, c10::optional<Variable> mask, Variable status,
                               int64_t max_len, double scale) {
    const c10::cuda::CUDAGuard guard(q.device());
    Tensors r;
    AT_DISPATCH_FLOATING_TYPES(q.scalar_type(), "structure attention second derivative", [&] {
      r = second_typed<scalar_t>(rows(a), rows(b), rows(c), go, q, k, v, o, lse, ptr, mask, max_len, scale, status);
    });
    return {r[3], r[0], r[1], r[2]};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "structure_attention on CUDA differentiates twice, not three times");
  }
};

// (dq, dk, dv); its own derivative is the total one, through o and the row statistics too
struct AttentionGrad : torch::autograd::Function<AttentionGrad> {
  static variable_list forward(AutogradContext* ctx, Variable go, Variable q, Variable k, Variable v, Variable o, Variable lse,
                               Variable ptr, c10::optional<Variable> mask, Variable status, int64_t max_len, double scale) {
    ctx->save_for_backward({go, q, k, v, o, lse, ptr, mask.value_or(Variable())});
    ctx->saved_data["status"] = status;
    keep(ctx, {max_len, scale});
    return attention_backward(go, q, k, v, o, lse, ptr, mask, max_len, scale, status);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    auto r = AttentionSecond::apply(g[0], g[1], g[2], s[0], s[1], s[2], s[3], s[4], s[5], s[6], maybe(s[7]),
                                    ctx->saved_data["status"].toTensor(), kept(ctx).max_len, kept(ctx).scale);
    r.resize(11);
    return r;
  }
};

struct Attention : torch::autograd::Function<Attention> {
  static Variable forward(AutogradContext* ctx, Variable q, Variable k, Variable v, Variable ptr, c10::optional<Variable> mask,
                          Variable status, int64_t max_len, double scale) {
    auto r = attention_forward(q, k, v, ptr, mask, max_len, scale, true, status);
    ctx->save_for_backward({q, k, v, r[0], r[1], ptr, mask.value_or(Variable())});
    ctx->saved_data["status"] = status;
    keep(ctx, {max_len, scale});
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const auto set = kept(ctx);
    no_tangents("structure_attention", {g[0]});
    if (!torch::GradMode::is_enabled()) {              // no graph of this pass is asked for
      auto r = attention_backward(rows(g[0]), s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]), set.max_len, set.scale,
                                  ctx->saved_data["status"].toTensor());
      r.resize(8);
      return r;
    }
    // o without its graph: the second derivative holds what goes through it
    // (the gradient's rows are laid out here, where that is recorded: the copy belongs to the graph)
    auto r = AttentionGrad::apply(rows(g[0]), s[0], s[1], s[2], s[3].detach(), s[4], s[5], maybe(s[6]),
                                  ctx->saved_data["status"].toTensor(), set.max_len, set.scale);
    r.resize(8);
    return r;
  }
};

// The arguments are checked here, not in Python: for the smallest structures the call costs more than its kernel.
template <typename... A>
void require(bool ok, const A&... what) {
  if (!ok) throw pybind11::value_error(c10::str(what...));
}
template <typename... A>
void require_type(bool ok, const A&... what) {
  if (!ok) throw pybind11::type_error(c10::str(what...));
}
bool floating(const torch::Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kFloat64; }

torch::Tensor structure_attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor ptr,
                                  c10::optional<int64_t> max_len, c10::optional<double> scale, c10::optional<torch::Tensor> mask,
                                  const torch::Tensor& status) {
  require(q.dim() == 3, "q must be (atoms, heads, width), got ", q.sizes());
  require(k.dim() == 3 && v.dim() == 3, "k and v must be (atoms, key heads, width), got ", k.sizes(), " and ", v.sizes());
  require_type(floating(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() &&
                   v.device() == q.device(),
               "q, k and v must all be float32 or all float64 on one device, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
               v.scalar_type());
  const int64_t n = q.size(0), h = q.size(1), d = q.size(2);
  require(k.size(0) == n && k.size(2) == d && v.sizes() == k.sizes(), "k and v must be (", n, ", key heads, ", d, "), got ", k.sizes(),
          " and ", v.sizes());
  require(h > 0 && d > 0 && k.size(1) > 0 && h % k.size(1) == 0, "the ", k.size(1), " key heads must divide the ", h, " query heads");
  require(ptr.dim() == 1 && ptr.numel() >= 1 && ptr.scalar_type() == torch::kInt64 && ptr.device() == q.device(),
          "ptr must be int64 (structures + 1) on ", q.device(), ", got ", ptr.scalar_type(), " ", ptr.sizes(), " on ", ptr.device());
  require(!mask.has_value() || (mask->scalar_type() == torch::kBool && mask->dim() == 1 && mask->size(0) == n && mask->device() == q.device()),
          "key_mask must be bool (", n, ") on ", q.device());
  require(max_len.value_or(0) >= 0, "max_len must not be negative, got ", max_len.value_or(0));
  no_tangents("structure_attention", {q, k, v});
  not_traced("structure_attention");
  require(d <= 128, "head width ", d, ": the kernels take up to 128");
  const int64_t most = max_len.value_or(n);
  const double f = scale.value_or(1.0 / std::sqrt((double)d));
  q = rows(q); k = rows(k); v = rows(v);
  ptr = ptr.contiguous();
  if (mask.has_value()) mask = mask->contiguous();
  if (torch::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return Attention::apply(q, k, v, ptr, mask, status, most, f);
  return attention_forward(q, k, v, ptr, mask, most, f, false, status)[0];
}

// x (outer, shared, inner) contiguous; rng int64 (seed, offset) on x's device
torch::Tensor dropout_raw(const torch::Tensor& x, int64_t outer, int64_t shared, int64_t inner, double p, const torch::Tensor& rng) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.numel() == outer * shared * inner, "counter_dropout: contiguous CUDA tensor");
  TORCH_CHECK(rng.device() == x.device() && rng.scalar_type() == torch::kInt64 && rng.numel() == 2 && rng.is_contiguous(),
              "counter_dropout: rng must be two int64 numbers on ", x.device());
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "counter_dropout: p in [0, 1]");
  TORCH_CHECK(shared < (1 << 30), "counter_dropout: too many shared copies");
  auto y = torch::empty_like(x);
  if (x.numel() == 0) return y;
  const auto s = at::cuda::getCurrentCUDAStream();
  AT_DISPATCH_FLOATING_TYPES(x.scalar_type(), "counter_dropout", [&] {
    XNN_OK(counter_dropout<scalar_t>(outer, shared, inner, p, rng.data_ptr<int64_t>(), x.data_ptr<scalar_t>(),
                                     y.data_ptr<scalar_t>(), s));
  });
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Variable forward(AutogradContext* ctx, Variable x, Variable rng, int64_t outer, int64_t shared, int64_t inner, double p) {
    ctx->save_for_backward({rng});
    ctx->saved_data["sizes"] = std::vector<int64_t>{outer, shared, inner};
    ctx->saved_data["p"] = p;
    return dropout_raw(x, outer, shared, inner, p, rng);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto n = ctx->saved_data["sizes"].toIntVector();
    no_tangents("counter_dropout", {g[0]});
    if (!torch::GradMode::is_enabled())
      return {dropout_raw(g[0].contiguous(), n[0], n[1], n[2], ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0]),
              Variable(), Variable(), Variable(), Variable(), Variable()};
    return {Dropout::apply(g[0].contiguous(), ctx->get_saved_variables()[0], n[0], n[1], n[2], ctx->saved_data["p"].toDouble()),
            Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};

// the sizes in front of, in and behind the dimensions that share a mask entry
std::array<int64_t, 3> shared_sizes(const torch::Tensor& x, const std::vector<int64_t>& shared) {
  std::array<int64_t, 3> n{1, 1, 1};
  if (shared.empty()) return {x.numel(), 1, 1};
  uint64_t set = 0;
  for (const int64_t s : shared) {
    require(s >= -x.dim() && s < x.dim() && x.dim() <= 64, "shared dimension ", s, " of a tensor with ", x.dim(), " dimensions");
    set |= 1ull << (s < 0 ? s + x.dim() : s);
  }
  int stage = 0;
  for (int64_t i = 0; i < x.dim(); ++i) {
    if (x.size(i) == 1) continue;
    if (set >> i & 1) {
      require(stage < 2, "the shared dimensions ", shared, " of shape ", x.sizes(), " must be neighbours");
      stage = 1;
    } else if (stage == 1) {
      stage = 2;
    }
    n[stage] *= x.size(i);
  }
  return n;
}

torch::Tensor dropout_op(torch::Tensor x, double p, torch::Tensor rng, const std::vector<int64_t>& shared) {
  require_type(floating(x), "counter_dropout takes float32 or float64, got ", x.scalar_type());
  require(p >= 0.0 && p <= 1.0, "the dropout probability must be in [0, 1], got ", p);
  require(rng.scalar_type() == torch::kInt64 && rng.dim() == 1 && rng.size(0) == 2 && rng.device() == x.device(),
          "rng must be two int64 numbers (seed, offset) on ", x.device());
  no_tangents("counter_dropout", {x});
  not_traced("counter_dropout");
  const auto n = shared_sizes(x, shared);
  x = x.contiguous();
  rng = rng.contiguous();
  if (torch::GradMode::is_enabled() && x.requires_grad()) return Dropout::apply(x, rng, n[0], n[1], n[2], p);
  return dropout_raw(x, n[0], n[1], n[2], p, rng);
}

void check_ids(const torch::Tensor& ids, const torch::Tensor& like) {
  TORCH_CHECK(ids.device() == like.device() && ids.is_contiguous() &&
                  (ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32),
              "embedding_lookup: ids must be contiguous int64 or int32 on ", like.device());
  TORCH_CHECK(ids.numel() < (1 << 30), "embedding_lookup: fewer than 2^30 ids");
}

torch::Tensor lookup_raw(const torch::Tensor& table, const torch::Tensor& ids, double scale) {
  const c10::cuda::CUDAGuard guard(table.device());
  TORCH_CHECK(table.is_cuda() && table.dim() == 2 && table.is_contiguous() && table.size(0) < (1 << 30) &&
                  table.size(1) < (1 << 20), "embedding_lookup: table (rows, width), contiguous on a CUDA device");
  check_ids(ids, table);
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  auto out = torch::empty(shape, table.options());
  if (out.numel() == 0) return out;
  const auto s = at::cuda::getCurrentCUDAStream();
  AT_DISPATCH_FLOATING_TYPES(table.scalar_type(), "embedding_lookup", [&] {
    if (ids.scalar_type() == torch::kInt64)
      XNN_OK((embedding_lookup<scalar_t, int64_t>(ids.numel(), table.size(0), (int)table.size(1), table.data_ptr<scalar_t>(),
                                                  ids.data_ptr<int64_t>(), scale, out.data_ptr<scalar_t>(), s)));
    else
      XNN_OK((embedding_lookup<scalar_t, int>(ids.numel(), table.size(0), (int)table.size(1), table.data_ptr<scalar_t>(),
                                              ids.data_ptr<int>(), scale, out.data_ptr<scalar_t>(), s)));
  });
  return out;
}

torch::Tensor lookup_grad_raw(const torch::Tensor& ids, const torch::Tensor& g, int64_t rows, double scale) {
  const c10::cuda::CUDAGuard guard(g.device());
  const int64_t N = ids.numel(), C = g.size(-1);
  TORCH_CHECK(g.is_cuda() && g.is_contiguous() && g.numel() == N * C && rows < (1 << 30) && C < (1 << 20),
              "embedding_lookup: gradient (ids, width), contiguous on a CUDA device");
  check_ids(ids, g);
  auto out = torch::empty({rows, C}, g.options());
  if (out.numel() == 0) return out;
  if (N == 0) return out.zero_();
  const auto s = at::cuda::getCurrentCUDAStream();
  auto ints = torch::empty({embedding_grad_ints(N, rows, C)}, g.options().dtype(torch::kInt32));
  auto parts = torch::empty({embedding_grad_partials(N, rows, C)}, g.options());
  AT_DISPATCH_FLOATING_TYPES(g.scalar_type(), "embedding_lookup gradient", [&] {
    if (ids.scalar_type() == torch::kInt64)
      XNN_OK((embedding_grad<scalar_t, int64_t>(N, rows, (int)C, ids.data_ptr<int64_t>(), g.data_ptr<scalar_t>(), scale,
                                                ints.data_ptr<int>(), parts.data_ptr<scalar_t>(), out.data_ptr<scalar_t>(), s)));
    else
      XNN_OK((embedding_grad<scalar_t, int>(N, rows, (int)C, ids.data_ptr<int>(), g.data_ptr<scalar_t>(), scale,
                                            ints.data_ptr<int>(), parts.data_ptr<scalar_t>(), out.data_ptr<scalar_t>(), s)));
  });
  return out;
}

// the lookup and its adjoint: each is the other's backward pass
struct LookupGrad : torch::autograd::Function<LookupGrad> {
  static Variable forward(AutogradContext* ctx, Variable g, Variable ids, int64_t rows, double scale);
  static variable_list backward(AutogradContext* ctx, variable_list t);
};
struct Lookup : torch::autograd::Function<Lookup> {
  static Variable forward(AutogradContext* ctx, Variable table, Variable ids, double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    return lookup_raw(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_tangents("embedding_lookup", {g[0]});
    if (!torch::GradMode::is_enabled())
      return {lookup_grad_raw(ctx->get_saved_variables()[0], g[0].contiguous(), ctx->saved_data["rows"].toInt(),
                              ctx->saved_data["scale"].toDouble()), Variable(), Variable()};
    return {LookupGrad::apply(g[0].contiguous(), ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                              ctx->saved_data["scale"].toDouble()), Variable(), Variable()};
  }
};
Variable LookupGrad::forward(AutogradContext* ctx, Variable g, Variable ids, int64_t rows, double scale) {
  ctx->save_for_backward({ids});
  ctx->saved_data["scale"] = scale;
  return lookup_grad_raw(ids, g, rows, scale);
}
variable_list LookupGrad::backward(AutogradContext* ctx, variable_list t) {
  return {Lookup::apply(t[0].contiguous(), ctx->get_saved_variables()[0], ctx->saved_data["scale"].toDouble()),
          Variable(), Variable(), Variable()};
}

torch::Tensor lookup_op(torch::Tensor table, torch::Tensor ids, double scale) {
  require_type(table.dim() == 2 && floating(table), "table must be (rows, width) float32 or float64, got ", table.scalar_type(), " ",
               table.sizes());
  require_type(ids.scalar_type() == torch::kInt64 || ids.scalar_type() == torch::kInt32, "ids must be int64 or int32, got ",
               ids.scalar_type());
  require(ids.device() == table.device(), "table on ", table.device(), ", ids on ", ids.device());
  no_tangents("embedding_lookup", {table});
  not_traced("embedding_lookup");
  table = table.contiguous();
  ids = ids.contiguous();
  if (torch::GradMode::is_enabled() && table.requires_grad()) return Lookup::apply(table, ids, scale);
  return lookup_raw(table, ids, scale);
}

}  // namespace

void register_transformer(pybind11::module& m) {
  m.def("structure_attention", &structure_attention);
  m.def("counter_dropout", &dropout_op);
  m.def("embedding_lookup", &lookup_op);
}
