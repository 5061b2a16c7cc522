// kat_torch.cpp — the q/k norm and the position biases as torch operators with their autograd nodes
// (libkat_torch.so, loaded by _native.ops()).
//
// Everything is computed by libkat_rational.so through its C entries, whose addresses kat_torch_bind
// takes.  What is here checks the arguments, allocates outputs, fills the entries' arguments and is the
// node of the backward pass.  It is C++ because these calls are short: a forward and backward pass of a
// 197-token grid bias takes its kernels 9 us and the call 67, 94 with the same nodes in Python (packed q/k
// norm of the ViT-B/16 block at batch 128: 97 and 156; one token's, forward alone: 11 and 21, and 14 with
// the checks in Python).

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "kat_position_bias.h"
#include "kat_qk_norm_rope.h"
#include "kat_rational.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Entries {
  decltype(&kat_rational_strerror) strerror;
  decltype(&kat_qk_norm_rope_fwd) qk_fwd;
  decltype(&kat_qk_norm_rope_bwd_workspace_bytes) qk_bwd_bytes;
  decltype(&kat_qk_norm_rope_bwd) qk_bwd;
  decltype(&kat_distance_bias_fwd) distance_fwd;
  decltype(&kat_distance_bias_bwd_workspace_bytes) distance_bwd_bytes;
  decltype(&kat_distance_bias_bwd) distance_bwd;
  decltype(&kat_index_bias_fwd) index_fwd;
  decltype(&kat_index_bias_bwd_workspace_bytes) index_bwd_bytes;
  decltype(&kat_index_bias_bwd) index_bwd;
};
Entries entries{};

void check(const char* name, int status) {
  TORCH_CHECK(status == KAT_OK, name, " failed: ", entries.strerror(status), " (status ", status, ")");
}

int32_t code_of(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return KAT_DTYPE_F32;
    case at::kHalf: return KAT_DTYPE_F16;
    case at::kBFloat16: return KAT_DTYPE_BF16;
    default: TORCH_CHECK(false, "expected float32, float16 or bfloat16, got ", type);
  }
}
at::ScalarType type_of(int64_t code) {
  return code == KAT_DTYPE_F32 ? at::kFloat : code == KAT_DTYPE_F16 ? at::kHalf : at::kBFloat16;
}

// What an operator takes, checked here too: torch.ops reaches it past the Python functions.
bool known_type(at::ScalarType type) {
  return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}
// Its values lie where it says (not so in a subclass that wraps other tensors).
bool plain(const Tensor& t) {
  return t.layout() == at::kStrided && !t._is_zerotensor() &&
         !t.unsafeGetTensorImpl()->is_python_dispatch();
}
bool whole(const Tensor& t, const Tensor& like) {
  return plain(t) && t.device() == like.device() && t.is_contiguous();
}
// `n` values of `type`, one after the other, where `like` is.
bool run_of(const Tensor& t, const Tensor& like, at::ScalarType type, int64_t n) {
  return t.scalar_type() == type && t.numel() == n && whole(t, like);
}
// The tensor with its values as they lie in memory (a conjugate's imaginary part is a view whose values
// are still to be negated).
Tensor settled(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor settled(const std::optional<Tensor>& t) { return t ? settled(*t) : Tensor(); }
void need_cuda(const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), name, ": expected CUDA tensors, got ", t.device());
}

// The current stream of a tensor's device, which is the current device meanwhile.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

Tensor bytes_like(const Tensor& t, size_t bytes) {
  return at::empty({int64_t(bytes)}, t.options().dtype(at::kByte));
}

// There is no forward-mode derivative: a tangent raises, also where no gradient is wanted.
void refuse_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                              "this operator has no forward-mode derivative");
}

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) refuse_tangent(*t);
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients have no gradient: under create_graph they hang on a node that says so.
struct Once : Function<Once> {
  static Tensor forward(AutogradContext*, const Tensor& result, const Tensor&) {
    return result.alias();
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "this operator's gradient cannot be differentiated again");
  }
};
variable_list once(variable_list results, const variable_list& from) {
  for (const Tensor& anchor : from) refuse_tangent(anchor);
  if (!at::GradMode::is_enabled()) return results;
  for (const Tensor& anchor : from) {
    if (!anchor.defined() || !anchor.requires_grad()) continue;
    for (Tensor& r : results)
      if (r.defined()) r = Once::apply(r, anchor);
    break;
  }
  return results;
}

// ---------------------------------------------------------------------------
// Norm of queries and keys with the rotation.
// ---------------------------------------------------------------------------

using Maybe = std::optional<Tensor>;
Maybe given(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

struct Rope {   // undefined tensors: none
  Tensor cos, sin, positions;
  double eps;
  bool interleaved;
};

void check_rope(const char* name, const Tensor& x, int64_t head_dim, const Tensor& q_weight,
                const Tensor& k_weight, const Rope& rope) {
  TORCH_CHECK(known_type(x.scalar_type()) && plain(x), name,
              ": queries and keys must be dense float32, float16 or bfloat16");
  TORCH_CHECK(head_dim >= 1 && head_dim <= 1024, name, ": head size must be 1..1024, got ", head_dim);
  for (const Tensor* w : {&q_weight, &k_weight})
    TORCH_CHECK(!w->defined() || (known_type(w->scalar_type()) && w->dim() == 1 &&
                                  w->numel() == head_dim && whole(*w, x)),
                name, ": a weight must be a contiguous [", head_dim, "] on ", x.device());
  TORCH_CHECK(!q_weight.defined() || !k_weight.defined() ||
                  q_weight.scalar_type() == k_weight.scalar_type(),
              name, ": the weights' types differ");
  TORCH_CHECK(rope.cos.defined() == rope.sin.defined(), name, ": cos and sin come together");
  if (!rope.cos.defined()) {
    TORCH_CHECK(!rope.positions.defined(), name, ": positions without a table");
    return;
  }
  TORCH_CHECK(rope.cos.dim() == 2 && rope.cos.sizes() == rope.sin.sizes() &&
                  2 * rope.cos.size(1) <= head_dim &&
                  run_of(rope.cos, x, at::kFloat, rope.cos.numel()) &&
                  run_of(rope.sin, x, at::kFloat, rope.cos.numel()) && !rope.cos.requires_grad() &&
                  !rope.sin.requires_grad(),
              name, ": cos and sin must be contiguous float32 [rows, at most ", head_dim / 2, "] on ",
              x.device(), ", without a gradient");
  if (rope.positions.defined()) {
    TORCH_CHECK(rope.positions.scalar_type() == at::kLong && plain(rope.positions) &&
                    rope.positions.device() == x.device() && rope.positions.dim() == 2 &&
                    rope.positions.size(0) == x.size(0) && rope.positions.size(1) == x.size(1),
                name, ": positions must be int64 [", x.size(0), ", ", x.size(1), "] on ", x.device());
  } else {
    TORCH_CHECK(rope.cos.size(0) >= x.size(1), name, ": ", x.size(1), " tokens, and a table of ",
                rope.cos.size(0), " rows");
  }
}

const void* pointer(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// The same values with a head's D values one after the other.
Tensor heads_of(const Tensor& t_in) {
  const Tensor t = settled(t_in);
  return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous();
}

kat_head_problem problem_of(int64_t batch, int64_t tokens, int64_t head_dim, at::ScalarType type,
                            const Tensor& q_weight, const Tensor& k_weight, const Rope& rope) {
  kat_head_problem p{};
  p.batch = batch;
  p.tokens = tokens;
  p.head_dim = int32_t(head_dim);
  p.dtype = code_of(type);
  const Tensor& weight = q_weight.defined() ? q_weight : k_weight;
  p.weight_dtype = weight.defined() ? code_of(weight.scalar_type()) : 0;
  p.eps = float(rope.eps);
  if (rope.cos.defined()) {
    p.rot_dim = int32_t(2 * rope.cos.size(1));
    p.interleaved = rope.interleaved;
    p.cos_table = rope.cos.const_data_ptr<float>();
    p.sin_table = rope.sin.const_data_ptr<float>();
    p.table_rows = rope.cos.size(0);
    if (rope.positions.defined()) {
      p.positions = rope.positions.const_data_ptr<int64_t>();
      p.position_stride[0] = rope.positions.stride(0);
      p.position_stride[1] = rope.positions.stride(1);
    }
  }
  return p;
}

struct Strides {
  int64_t batch, token, head;
};
Strides strides_of(const Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }
void put(int64_t (&to)[3], const Strides& s) {
  to[0] = s.batch;
  to[1] = s.token;
  to[2] = s.head;
}
// `offset` elements behind a tensor's first, where it has any.
const void* behind(const Tensor& t, int64_t offset) {
  const char* p = static_cast<const char*>(t.const_data_ptr());
  return p == nullptr ? nullptr : p + offset * int64_t(t.element_size());
}

kat_head_stream stream_of(const void* x, const Strides& xs, const void* out, const Strides& os,
                          const Tensor& weight, int64_t heads) {
  kat_head_stream s{};
  s.x = x;
  put(s.x_stride, xs);
  s.out = const_cast<void*>(out);
  put(s.out_stride, os);
  s.weight = pointer(weight);
  s.heads = int32_t(heads);
  return s;
}
void put_grad(kat_head_stream& s, const Tensor& dy, const Tensor& dweight) {
  s.dy = dy.const_data_ptr();
  put(s.dy_stride, strides_of(dy));
  s.dweight = dweight.defined() ? dweight.mutable_data_ptr<float>() : nullptr;
}

Tensor dweight_of(const Tensor& weight) {
  return weight.defined() && weight.requires_grad()
             ? at::empty(weight.sizes(), weight.options().dtype(at::kFloat).requires_grad(false))
             : Tensor();
}
Tensor as(const Tensor& grad, const Tensor& like) {
  return grad.defined() ? grad.to(like.scalar_type()) : grad;
}

void run_backward(const kat_head_problem& p, const kat_head_stream* streams, int count,
                  const Tensor& like) {
  const On on(like);
  const size_t bytes = entries.qk_bwd_bytes(p.head_dim, count, like.device().index());
  TORCH_CHECK(bytes > 0, "kat_qk_norm_rope_bwd_workspace_bytes returned 0");
  const Tensor ws = bytes_like(like, bytes);
  check("kat_qk_norm_rope_bwd",
        entries.qk_bwd(&p, streams, count, ws.mutable_data_ptr(), bytes, on.stream));
}

variable_list saved_of(const Tensor& a, const Tensor& b, const Tensor& q_weight,
                       const Tensor& k_weight, const Rope& rope) {
  return {a, b, q_weight, k_weight, rope.cos, rope.sin, rope.positions};
}
Rope rope_of(AutogradContext* ctx, const variable_list& saved) {
  return {saved[4], saved[5], saved[6], ctx->saved_data["eps"].toDouble(),
          ctx->saved_data["interleaved"].toBool()};
}
void keep_rope(AutogradContext* ctx, const Rope& rope) {
  ctx->saved_data["eps"] = rope.eps;
  ctx->saved_data["interleaved"] = rope.interleaved;
}

variable_list qk_forward(const Tensor& q, const Tensor& k, const Tensor& q_weight,
                         const Tensor& k_weight, const Rope& rope) {
  const On on(q);
  const Tensor out_q = at::empty(q.sizes(), q.options().requires_grad(false));
  const Tensor out_k = at::empty(k.sizes(), k.options().requires_grad(false));
  const auto p = problem_of(q.size(0), q.size(1), q.size(3), q.scalar_type(), q_weight, k_weight, rope);
  const kat_head_stream s[2] = {
      stream_of(q.const_data_ptr(), strides_of(q), out_q.const_data_ptr(), strides_of(out_q), q_weight,
                q.size(2)),
      stream_of(k.const_data_ptr(), strides_of(k), out_k.const_data_ptr(), strides_of(out_k), k_weight,
                k.size(2))};
  check("kat_qk_norm_rope_fwd", entries.qk_fwd(&p, s, 2, on.stream));
  return {out_q, out_k};
}

struct QkNormRope : Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in,
                               const Maybe& q_maybe, const Maybe& k_maybe, const Rope& rope) {
    const Tensor q = heads_of(q_in), k = heads_of(k_in);
    const Tensor q_weight = q_maybe.value_or(Tensor()), k_weight = k_maybe.value_or(Tensor());
    ctx->save_for_backward(saved_of(q, k, q_weight, k_weight, rope));
    keep_rope(ctx, rope);
    return qk_forward(q, k, q_weight, k_weight, rope);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &q_weight = saved[2], &k_weight = saved[3];
    const Rope rope = rope_of(ctx, saved);
    const Tensor gq = heads_of(grads[0]), gk = heads_of(grads[1]);
    const Tensor dq = at::empty(q.sizes(), q.options().requires_grad(false));
    const Tensor dk = at::empty(k.sizes(), k.options().requires_grad(false));
    const Tensor dwq = dweight_of(q_weight), dwk = dweight_of(k_weight);
    const auto p =
        problem_of(q.size(0), q.size(1), q.size(3), q.scalar_type(), q_weight, k_weight, rope);
    kat_head_stream s[2] = {
        stream_of(q.const_data_ptr(), strides_of(q), dq.const_data_ptr(), strides_of(dq), q_weight,
                  q.size(2)),
        stream_of(k.const_data_ptr(), strides_of(k), dk.const_data_ptr(), strides_of(dk), k_weight,
                  k.size(2))};
    put_grad(s[0], gq, dwq);
    put_grad(s[1], gk, dwk);
    run_backward(p, s, 2, q);
    return once({dq, dk, as(dwq, q_weight), as(dwk, k_weight), Tensor()},
                {grads[0], grads[1], q, k, q_weight, k_weight});
  }
};

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k,
                                        const Maybe& q_weight,
                                        const Maybe& k_weight,
                                        const Maybe& cos,
                                        const Maybe& sin,
                                        const Maybe& positions, double eps,
                                        bool interleaved) {
  const Tensor wq = settled(q_weight), wk = settled(k_weight);
  const Rope rope{settled(cos), settled(sin), settled(positions), eps, interleaved};
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                  q.size(3) == k.size(3) && q.scalar_type() == k.scalar_type() &&
                  q.device() == k.device() && plain(k),
              "qk_norm_rope: expected q [B, L, Hq, D] and k [B, L, Hk, D] of one type on one device");
  check_rope("qk_norm_rope", q, q.size(3), wq, wk, rope);
  need_cuda("qk_norm_rope", q);
  const variable_list out = wants_grad({&q, &k, &wq, &wk, &rope.cos, &rope.sin})
                                ? QkNormRope::apply(q, k, given(wq), given(wk), rope)
                                : qk_forward(heads_of(q), heads_of(k), wq, wk, rope);
  return {out[0], out[1]};
}

Tensor packed_of(const Tensor& qkv_in) {
  const Tensor qkv = settled(qkv_in);
  return qkv.stride(2) == 1 || qkv.size(2) == 1 ? qkv : qkv.contiguous();
}

// q', k' and v, a view of x.
variable_list qkv_forward(const Tensor& x, int64_t hq, int64_t hk, const Tensor& q_weight,
                          const Tensor& k_weight, const Rope& rope) {
  const On on(x);
  const int64_t B = x.size(0), L = x.size(1), D = x.size(2) / (hq + 2 * hk);
  const auto options = x.options().requires_grad(false);
  const Tensor out_q = at::empty({B, L, hq, D}, options), out_k = at::empty({B, L, hk, D}, options);
  const Strides xs{x.stride(0), x.stride(1), D};
  const auto p = problem_of(B, L, D, x.scalar_type(), q_weight, k_weight, rope);
  const kat_head_stream s[2] = {
      stream_of(behind(x, 0), xs, out_q.const_data_ptr(), strides_of(out_q), q_weight, hq),
      stream_of(behind(x, hq * D), xs, out_k.const_data_ptr(), strides_of(out_k), k_weight, hk)};
  check("kat_qk_norm_rope_fwd", entries.qk_fwd(&p, s, 2, on.stream));
  return {out_q, out_k,
          x.as_strided({B, L, hk, D}, {x.stride(0), x.stride(1), D, 1},
                       x.storage_offset() + (hq + hk) * D)};
}

struct QkvNormRope : Function<QkvNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Maybe& q_maybe,
                               const Maybe& k_maybe, int64_t hq, int64_t hk, const Rope& rope) {
    const Tensor x = packed_of(qkv);
    const Tensor q_weight = q_maybe.value_or(Tensor()), k_weight = k_maybe.value_or(Tensor());
    ctx->save_for_backward(saved_of(x, Tensor(), q_weight, k_weight, rope));
    keep_rope(ctx, rope);
    ctx->saved_data["hq"] = hq;
    ctx->saved_data["hk"] = hk;
    return qkv_forward(x, hq, hk, q_weight, k_weight, rope);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &q_weight = saved[2], &k_weight = saved[3];
    const Rope rope = rope_of(ctx, saved);
    const int64_t hq = ctx->saved_data["hq"].toInt(), hk = ctx->saved_data["hk"].toInt();
    const Tensor gq = heads_of(grads[0]), gk = heads_of(grads[1]), gv = heads_of(grads[2]);
    const int64_t width = x.size(2), L = x.size(1), D = width / (hq + 2 * hk);
    const Tensor dx = at::empty(x.sizes(), x.options().requires_grad(false));
    const Tensor dwq = dweight_of(q_weight), dwk = dweight_of(k_weight);
    const Strides xs{x.stride(0), x.stride(1), D}, os{L * width, width, D};
    const auto p = problem_of(x.size(0), L, D, x.scalar_type(), q_weight, k_weight, rope);
    kat_head_stream s[3] = {
        stream_of(behind(x, 0), xs, behind(dx, 0), os, q_weight, hq),
        stream_of(behind(x, hq * D), xs, behind(dx, hq * D), os, k_weight, hk),
        stream_of(nullptr, {0, 0, 0}, behind(dx, (hq + hk) * D), os, Tensor(), hk)};
    put_grad(s[0], gq, dwq);
    put_grad(s[1], gk, dwk);
    put_grad(s[2], gv, Tensor());
    run_backward(p, s, 3, x);
    return once({dx, as(dwq, q_weight), as(dwk, k_weight), Tensor(), Tensor(), Tensor()},
                {grads[0], grads[1], grads[2], x, q_weight, k_weight});
  }
};

std::tuple<Tensor, Tensor, Tensor> qkv_norm_rope(const Tensor& qkv, int64_t q_heads, int64_t k_heads,
                                                 const Maybe& q_weight,
                                                 const Maybe& k_weight,
                                                 const Maybe& cos,
                                                 const Maybe& sin,
                                                 const Maybe& positions, double eps,
                                                 bool interleaved) {
  const Tensor wq = settled(q_weight), wk = settled(k_weight);
  const Rope rope{settled(cos), settled(sin), settled(positions), eps, interleaved};
  constexpr int64_t most = int64_t(1) << 31;
  TORCH_CHECK(qkv.dim() == 3 && q_heads >= 1 && k_heads >= 1 && q_heads < most && k_heads < most &&
                  qkv.size(2) > 0 && qkv.size(2) % (q_heads + 2 * k_heads) == 0,
              "qkv_norm_rope: expected [B, L, (q_heads + 2 k_heads) D]");
  check_rope("qkv_norm_rope", qkv, qkv.size(2) / (q_heads + 2 * k_heads), wq, wk, rope);
  need_cuda("qkv_norm_rope", qkv);
  const variable_list out = wants_grad({&qkv, &wq, &wk, &rope.cos, &rope.sin})
                                ? QkvNormRope::apply(qkv, given(wq), given(wk), q_heads, k_heads, rope)
                                : qkv_forward(packed_of(qkv), q_heads, k_heads, wq, wk, rope);
  return {out[0], out[1], out[2]};
}

// ---------------------------------------------------------------------------
// Position biases.
// ---------------------------------------------------------------------------

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// Rows padded to multiples of 8, and their lk columns as a tensor of its own: autograd does not know it
// as a view, which could not be changed in place outside the node that made it.
std::pair<Tensor, Tensor> rows_of(const Tensor& table, int64_t lq, int64_t lk, int64_t type) {
  const Tensor out = at::empty({table.size(1), lq, round8(lk)},
                               table.options().dtype(type_of(type)).requires_grad(false));
  if (lk % 8 == 0) return {out, out};
  const at::AutoDispatchBelowADInplaceOrView no_views;
  return {out, out.narrow(2, 0, lk)};
}
Tensor dtable_of(const Tensor& grad, int64_t buckets, at::ScalarType type) {
  return at::empty({buckets, grad.size(0)}, grad.options().dtype(type).requires_grad(false));
}

constexpr int64_t kMaxLength = (int64_t(1) << 31) - 64;   // as the entries have it

// The values of a plan are those DistanceBuckets or IndexBuckets made; its sizes are checked.
void check_table(const char* name, const Tensor& table, int64_t buckets, int64_t lq, int64_t lk,
                 int64_t type) {
  TORCH_CHECK(table.dim() == 2 && plain(table) && known_type(table.scalar_type()) && buckets >= 1 &&
                  table.size(0) == buckets && buckets <= (int64_t(1) << 24) && table.size(1) <= 65535,
              name, ": expected a dense float32, float16 or bfloat16 table [", buckets, ", heads]");
  TORCH_CHECK(lq >= 0 && lk >= 0 && lq <= kMaxLength && lk <= kMaxLength, name,
              ": lengths must be 0..", kMaxLength, ", got ", lq, " and ", lk);
  TORCH_CHECK(type == KAT_DTYPE_F32 || type == KAT_DTYPE_F16 || type == KAT_DTYPE_BF16, name,
              ": unknown type ", type);
}

struct Distance {
  Tensor bucket_of, run_begin, run_end;
  int64_t buckets, reach, lq, lk, offset, causal, type;
};

Tensor distance_forward(const Tensor& table_in, const Distance& a) {
  const On on(table_in);
  const Tensor table = settled(table_in).contiguous();
  const auto out = rows_of(table, a.lq, a.lk, a.type);
  check("kat_distance_bias_fwd",
        entries.distance_fwd(table.const_data_ptr(), code_of(table.scalar_type()), int32_t(a.buckets),
                             int32_t(table.size(1)), a.bucket_of.const_data_ptr<int32_t>(),
                             int32_t(a.reach), a.lq, a.lk, a.offset, int32_t(a.causal),
                             out.first.mutable_data_ptr(), int32_t(a.type), on.stream));
  return out.second;
}

struct DistanceBias : Function<DistanceBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Distance& a) {
    ctx->saved_data["runs"] = std::vector<Tensor>{a.run_begin, a.run_end};
    ctx->saved_data["sizes"] = std::vector<int64_t>{a.buckets, a.lq, a.lk, a.offset, a.causal,
                                                    int64_t(table.scalar_type())};
    return distance_forward(table, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor grad = settled(grads[0]);
    const auto runs = ctx->saved_data["runs"].toTensorVector();
    const auto n = ctx->saved_data["sizes"].toIntVector();
    const On on(grad);
    const int32_t heads = int32_t(grad.size(0));
    const auto type = at::ScalarType(n[5]);
    const Tensor d = dtable_of(grad, n[0], type);
    const size_t bytes = entries.distance_bwd_bytes(heads, n[1], n[2]);
    const Tensor ws = bytes_like(grad, bytes);
    check("kat_distance_bias_bwd",
          entries.distance_bwd(grad.const_data_ptr(), code_of(grad.scalar_type()),
                               grad.strides().data(), int32_t(n[0]), heads,
                               runs[0].const_data_ptr<int32_t>(), runs[1].const_data_ptr<int32_t>(),
                               n[1], n[2], n[3], int32_t(n[4]), d.mutable_data_ptr(), code_of(type),
                               ws.mutable_data_ptr(), bytes, on.stream));
    return once({d, Tensor()}, {grad});
  }
};

Tensor distance_bias(const Tensor& table, at::TensorList plan, int64_t buckets, int64_t reach,
                     int64_t lq, int64_t lk, int64_t offset, bool causal, int64_t type) {
  check_table("distance_bias", table, buckets, lq, lk, type);
  TORCH_CHECK(offset >= -kMaxLength && offset <= kMaxLength, "distance_bias: |offset| must be 0..",
              kMaxLength, ", got ", offset);
  TORCH_CHECK(plan.size() == 3 && reach >= 0 && reach <= (int64_t(1) << 24) &&
                  run_of(plan[0], table, at::kInt, 2 * reach + 1) &&
                  run_of(plan[1], table, at::kInt, buckets) && run_of(plan[2], table, at::kInt, buckets),
              "distance_bias: the plan has another reach, number of buckets or device");
  need_cuda("distance_bias", table);
  const Distance a{plan[0], plan[1], plan[2], buckets, reach, lq, lk, offset, causal, type};
  return wants_grad({&table}) ? DistanceBias::apply(table, a) : distance_forward(table, a);
}

struct Index {
  at::TensorList plan;   // index, cells, padded_cells, seg_begin, slab_begin, seg_place, bucket_begin
  int64_t buckets, lq, lk, slab_rows, slabs, segments, type;
};

Tensor index_forward(const Tensor& table_in, const Index& a) {
  const On on(table_in);
  const Tensor table = settled(table_in).contiguous();
  const auto out = rows_of(table, a.lq, a.lk, a.type);
  check("kat_index_bias_fwd",
        entries.index_fwd(table.const_data_ptr(), code_of(table.scalar_type()), int32_t(a.buckets),
                          int32_t(table.size(1)), a.plan[0].const_data_ptr<int32_t>(), a.lq, a.lk,
                          out.first.mutable_data_ptr(), int32_t(a.type), on.stream));
  return out.second;
}

struct IndexBias : Function<IndexBias> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Index& a) {
    ctx->saved_data["plan"] = a.plan.vec();
    ctx->saved_data["sizes"] = std::vector<int64_t>{a.buckets, a.lq, a.lk, a.slab_rows, a.slabs,
                                                    a.segments, int64_t(table.scalar_type())};
    return index_forward(table, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor grad = settled(grads[0]);
    const auto plan = ctx->saved_data["plan"].toTensorVector();
    const auto n = ctx->saved_data["sizes"].toIntVector();
    const On on(grad);
    const int32_t heads = int32_t(grad.size(0));
    const auto type = at::ScalarType(n[6]);
    const Tensor d = dtable_of(grad, n[0], type);
    const size_t bytes = entries.index_bwd_bytes(heads, n[5]);
    const Tensor ws = bytes_like(grad, bytes);
    auto ints = [&](int i) { return plan[i].const_data_ptr<int32_t>(); };
    auto cells = [&](int i) { return static_cast<const uint16_t*>(plan[i].const_data_ptr()); };
    check("kat_index_bias_bwd",
          entries.index_bwd(grad.const_data_ptr(), code_of(grad.scalar_type()), grad.strides().data(),
                            int32_t(n[0]), heads, n[1], n[2], cells(1), cells(2), ints(3), n[5], ints(4),
                            n[4], int32_t(n[3]), ints(5), ints(6), d.mutable_data_ptr(), code_of(type),
                            ws.mutable_data_ptr(), bytes, on.stream));
    return once({d, Tensor()}, {grad});
  }
};

Tensor index_bias(const Tensor& table, at::TensorList plan, int64_t buckets, int64_t lq, int64_t lk,
                  int64_t slab_rows, int64_t slabs, int64_t segments, int64_t type) {
  check_table("index_bias", table, buckets, lq, lk, type);
  TORCH_CHECK(plan.size() == 7 && slabs >= 0 && segments >= 0 && slab_rows >= 1 &&
                  lk <= KAT_BIAS_SLAB_CELLS &&
                  run_of(plan[0], table, at::kInt, lq * round8(lk)) &&
                  run_of(plan[1], table, at::kUInt16, plan[1].numel()) &&
                  run_of(plan[2], table, at::kUInt16, plan[1].numel()) &&
                  run_of(plan[3], table, at::kInt, segments + 1) &&
                  run_of(plan[4], table, at::kInt, slabs + 1) &&
                  run_of(plan[5], table, at::kInt, segments) &&
                  run_of(plan[6], table, at::kInt, buckets + 1),
              "index_bias: the plan has another shape, number of buckets or device");
  need_cuda("index_bias", table);
  const Index a{plan, buckets, lq, lk, slab_rows, slabs, segments, type};
  return wants_grad({&table}) ? IndexBias::apply(table, a) : index_forward(table, a);
}

}  // namespace

// The addresses of libkat_rational.so's entries, in the order of `Entries`.
extern "C" __attribute__((visibility("default"))) void kat_torch_bind(const Entries* from) {
  entries = *from;
}

TORCH_LIBRARY(rational_kat_cu_b200, m) {
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, Tensor? sin, "
        "Tensor? positions, float eps, bool interleaved) -> (Tensor, Tensor)", &qk_norm_rope);
  m.def("qkv_norm_rope(Tensor(a) qkv, int q_heads, int k_heads, Tensor? q_weight, Tensor? k_weight, "
        "Tensor? cos, Tensor? sin, Tensor? positions, float eps, bool interleaved) -> "
        "(Tensor, Tensor, Tensor(a))", &qkv_norm_rope);
  m.def("distance_bias(Tensor table, Tensor[] plan, int buckets, int reach, int lq, int lk, int offset, "
        "bool causal, int type) -> Tensor", &distance_bias);
  m.def("index_bias(Tensor table, Tensor[] plan, int buckets, int lq, int lk, int slab_rows, int slabs, "
        "int segments, int type) -> Tensor", &index_bias);
}
