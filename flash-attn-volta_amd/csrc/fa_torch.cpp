// Autograd nodes of flash_attn / flash_attn_gqa, apply_rotary_qk and
// apply_rotary_positions in C++
// (Python module flash_attn_volta._fa_torch), a client of the C ABI in
// fa_mi355x.h.
//
// The reference's autograd.Function (flash_attn_volta/autograd.py:19-59)
// is Python, and so is this package's (autograd.py).  A Python backward
// node makes torch's autograd engine thread take the GIL while the thread
// that called backward() waits for it, a hand-off that costs about as much
// host time as the whole fwd+bwd launch work of a small config.  This node
// runs its backward in C++ without the GIL.  Python keeps the argument
// checks and the per-signature launch plan (forward.py); a plan handed
// here (make_plan) holds the sizes, strides, scale and workspace sizes the
// two C calls need, and attn() runs the forward and records the node.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <optional>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "fa_mi355x.h"

// Weak, so that the module still loads beside a library of another ABI
// version without them, as far as the version check below.
extern "C" {
__attribute__((weak)) decltype(fa_rope_qk_fwd) fa_rope_qk_fwd;
__attribute__((weak)) decltype(fa_rope_qk_bwd) fa_rope_qk_bwd;
__attribute__((weak)) decltype(fa_rope_qk_workspace_bytes) fa_rope_qk_workspace_bytes;
__attribute__((weak)) decltype(fa_rotary) fa_rotary;
__attribute__((weak)) decltype(fa_paged_append) fa_paged_append;
__attribute__((weak)) decltype(fa_paged_read) fa_paged_read;
__attribute__((weak)) decltype(fa_paged_attn) fa_paged_attn;
__attribute__((weak)) decltype(fa_paged_attn_workspace_bytes) fa_paged_attn_workspace_bytes;
}

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Launch arguments of one call signature.  Plans live until the process
// ends (deduplicated by content), so a node's plan pointer never dangles.
struct Plan {
  int B, Sq, Sk, H, Hk, D;
  int gqa, causal, dtype;
  float scale;
  int64_t q_st[4], k_st[4], v_st[4], o_st[4];   // kernel strides, 0 for size-1 dims
  int64_t dq_st[4], dk_st[4];                   // contiguous gradients
  size_t fwd_ws;                                // fa_fwd_ws workspace, 0: plain forward
  size_t ws_split, ws_plain;                    // backward workspace, split schedule or not
};

constexpr size_t kPlanInts = 9 + 24 + 3;

std::mutex g_mu;
std::map<std::vector<int64_t>, std::unique_ptr<Plan>> g_plans;
std::unordered_set<int64_t> g_handles;

int64_t make_plan(const std::vector<int64_t> &v, double scale) {
  TORCH_CHECK(v.size() == kPlanInts, "make_plan: expected ", kPlanInts, " integers, got ", v.size());
  std::vector<int64_t> key(v);
  const float s = static_cast<float>(scale);
  int32_t bits;
  std::memcpy(&bits, &s, sizeof bits);
  key.push_back(bits);
  std::lock_guard<std::mutex> lock(g_mu);
  auto it = g_plans.find(key);
  if (it != g_plans.end()) return reinterpret_cast<int64_t>(it->second.get());
  auto p = std::make_unique<Plan>();
  size_t i = 0;
  p->B = (int)v[i++]; p->Sq = (int)v[i++]; p->Sk = (int)v[i++];
  p->H = (int)v[i++]; p->Hk = (int)v[i++]; p->D = (int)v[i++];
  p->gqa = (int)v[i++]; p->causal = (int)v[i++]; p->dtype = (int)v[i++];
  for (int64_t *st : {p->q_st, p->k_st, p->v_st, p->o_st, p->dq_st, p->dk_st})
    for (int j = 0; j < 4; ++j) st[j] = v[i++];
  p->fwd_ws = (size_t)v[i++];
  p->ws_split = (size_t)v[i++];
  p->ws_plain = (size_t)v[i++];
  p->scale = s;
  const int64_t h = reinterpret_cast<int64_t>(p.get());
  g_handles.insert(h);
  g_plans.emplace(std::move(key), std::move(p));
  return h;
}

const Plan &plan_of(int64_t h) {
  std::lock_guard<std::mutex> lock(g_mu);
  TORCH_CHECK(g_handles.count(h), "flash_attn_volta._fa_torch: unknown plan handle");
  return *reinterpret_cast<const Plan *>(h);
}

void *stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

bool aligned(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// The kernels' strides of a (B, S, H, D) tensor they can read in place (unit
// D stride, the others non-negative multiples of 8 elements, 128 rows of a
// head within 31-bit byte offsets; `half_cols`, the attention kernels at 16
// columns: a whole head), 0 for size-1 dims, as the plan's; false for any
// other layout.
bool kernel_strides(const Tensor &t, int64_t (&st)[4], bool half_cols = false) {
  const int64_t *size = t.sizes().data(), *stride = t.strides().data();
  if (stride[3] != 1) return false;
  for (int i = 0; i < 3; ++i) {
    st[i] = size[i] == 1 ? 0 : stride[i];
    if (st[i] < 0 || (st[i] & 7) != 0) return false;
  }
  st[3] = 1;
  if (half_cols && (double)(size[1] - 1) * st[1] * 2 + 64 > INT32_MAX) return false;
  return 127 * st[1] * 2 + 2 * size[3] <= INT32_MAX;
}

// `t` as the kernels read it, its strides in `st`: itself where the layout and
// alignment allow, else a contiguous copy.
Tensor kernel_ready(const Tensor &t, int64_t (&st)[4], bool half_cols = false) {
  if (kernel_strides(t, st, half_cols) && aligned(t)) return t;
  Tensor c = t.clone(at::MemoryFormat::Contiguous);
  kernel_strides(c, st);
  return c;
}

// What a node saved may come back changed: hooks on saved tensors
// (torch.autograd.graph) return a tensor of their own, save_on_cpu for one a
// contiguous copy of any view.  The strides that a backward passes are
// therefore the returned tensor's; one of another shape, type or device than
// was saved is refused, as the kernels would read past its end.
void check_saved(const Tensor &t, at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  TORCH_CHECK(t.defined() && t.sizes() == sizes && t.scalar_type() == dtype &&
                  t.device() == device,
              "flash_attn_volta: a saved tensor came back with another shape, dtype or device");
}

void check(int rc, const char *where) {
  TORCH_CHECK(rc == FA_OK, where, ": ", fa_strerror(rc), " (status ", rc, ")");
}

struct FlashAttnFn : public torch::autograd::Function<FlashAttnFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                        int64_t handle, bool split) {
    const Plan &p = *reinterpret_cast<const Plan *>(handle);
    const c10::DeviceGuard guard(q.device());
    // (head_dim 16 runs as half of p.D = 32)
    Tensor out = at::empty({p.B, p.Sq, p.H, q.size(3)}, q.options());
    Tensor lse = at::empty({p.B, p.H, p.Sq}, q.options().dtype(at::kFloat));
    void *stream = stream_of(q);
    if (p.fwd_ws) {
      Tensor ws = at::empty({(int64_t)p.fwd_ws}, q.options().dtype(at::kByte));
      check(fa_fwd_ws(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                      lse.data_ptr<float>(), ws.data_ptr(), p.fwd_ws, p.B, p.Sq, p.Sk, p.H, p.Hk,
                      p.D, p.q_st, p.k_st, p.v_st, p.o_st, p.scale, p.causal, p.dtype, stream),
            "fa_fwd_ws");
    } else if (p.gqa) {
      check(fa_fwd_gqa(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                       lse.data_ptr<float>(), p.B, p.Sq, p.Sk, p.H, p.Hk, p.D, p.q_st, p.k_st,
                       p.v_st, p.o_st, p.scale, p.causal, p.dtype, stream),
            "fa_fwd_gqa");
    } else {
      check(fa_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr<float>(),
                   p.B, p.Sq, p.H, p.D, p.q_st, p.k_st, p.v_st, p.o_st, p.scale, p.causal, stream),
            "fa_fwd");
    }
    ctx->save_for_backward({q, k, v, out, lse});
    ctx->saved_data["plan"] = handle;
    ctx->saved_data["split"] = split;
    return out;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Plan &p = *reinterpret_cast<const Plan *>(ctx->saved_data["plan"].toInt());
    const bool split = ctx->saved_data["split"].toBool();
    // the engine hands dO over in out's shape, on its device
    const at::Device device = grads[0].device();
    const auto dtype = (p.dtype & ~FA_HALF_COLS) == FA_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
    const int64_t cols = grads[0].size(3);
    const c10::DeviceGuard guard(device);
    for (int i : {0, 3}) check_saved(s[i], {p.B, p.Sq, p.H, cols}, dtype, device);
    for (int i : {1, 2}) check_saved(s[i], {p.B, p.Sk, p.Hk, cols}, dtype, device);
    check_saved(s[4], {p.B, p.H, p.Sq}, at::kFloat, device);
    int64_t q_st[4], k_st[4], v_st[4], o_st[4], do_st[4];
    const bool half = cols != p.D;
    const Tensor q = kernel_ready(s[0], q_st, half), k = kernel_ready(s[1], k_st, half),
                 v = kernel_ready(s[2], v_st, half), out = kernel_ready(s[3], o_st, half);
    const Tensor lse = s[4].is_contiguous() && aligned(s[4])
                           ? s[4] : s[4].clone(at::MemoryFormat::Contiguous);
    // dO as the kernels read it: the forward's dtype, in place when its
    // layout allows (a model's transposed (B, H, S, D) gradient does: making
    // it contiguous cost 11 us of 113 at (8,1024,12,64)), 16-byte aligned
    const Tensor dout = kernel_ready(
        grads[0].scalar_type() == dtype ? grads[0] : grads[0].to(dtype), do_st, half);
    Tensor dq = at::empty({p.B, p.Sq, p.H, cols}, q.options());
    // separate allocations, as the Python path's
    Tensor dk = at::empty({p.B, p.Sk, p.Hk, cols}, q.options());
    Tensor dv = at::empty({p.B, p.Sk, p.Hk, cols}, q.options());
    const size_t nb = split ? p.ws_split : p.ws_plain;
    Tensor ws = at::empty({(int64_t)nb}, q.options().dtype(at::kByte));
    void *stream = stream_of(q);
    if (p.gqa) {
      check(fa_bwd_gqa(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                       lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                       ws.data_ptr(), nb, p.B, p.Sq, p.Sk, p.H, p.Hk, p.D, do_st, q_st,
                       k_st, v_st, o_st, p.dq_st, p.dk_st, p.dk_st, p.scale, p.causal,
                       p.dtype, stream),
            "fa_bwd_gqa");
    } else {
      check(fa_bwd(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                   lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                   ws.data_ptr(), nb, p.B, p.Sq, p.H, p.D, do_st, q_st, k_st, v_st,
                   o_st, p.dq_st, p.dk_st, p.dk_st, p.scale, p.causal, stream),
            "fa_bwd");
    }
    return {dq, dk, dv, Tensor(), Tensor()};
  }
};

// The forward of plan `handle` on q, k, v (whose shapes, strides, dtype and
// device the caller matched to the plan), recording the backward node when
// any input requires grad.  None when a data pointer is not 16-byte
// aligned: the caller then takes its general path.
std::optional<Tensor> attn(int64_t handle, const Tensor &q, const Tensor &k, const Tensor &v,
                           bool split) {
  plan_of(handle);
  if (!aligned(q) || !aligned(k) || !aligned(v)) return std::nullopt;
  return FlashAttnFn::apply(q, k, v, handle, split);
}

// The QK-norm + rotary prologue (rope.py's apply_rotary_qk) on tensors the
// kernels read in place.  A step of it is three kernels of some 45 us at
// (1, 4096, 32 / 8 heads, 128); a Python node around them took 178 us of host
// time a step.
using OptTensor = std::optional<Tensor>;

int dtype_of(const Tensor &t) {
  return t.scalar_type() == at::kHalf ? FA_DTYPE_F16 : FA_DTYPE_BF16;
}

const void *ptr_or_null(const OptTensor &t) { return t && t->defined() ? t->data_ptr() : nullptr; }

// (b, s) strides of a (1 or B, S, D) or (S, D) table, 0 for size-1 dims.
void table_strides(const Tensor &t, int64_t (&st)[2]) {
  const int64_t d = t.dim();
  st[0] = d == 2 || t.size(0) == 1 ? 0 : t.stride(0);
  st[1] = t.size(d - 2) == 1 ? 0 : t.stride(d - 2);
}

// A table that the kernels read in place, its strides in `st`: unit D stride,
// the others non-negative multiples of 8 elements, 16-byte aligned.
bool table_ready(const Tensor &t, int64_t (&st)[2]) {
  table_strides(t, st);
  return t.stride(t.dim() - 1) == 1 && st[0] >= 0 && st[1] >= 0 && st[0] % 8 == 0 &&
         st[1] % 8 == 0 && aligned(t);
}

struct RopeFn : public torch::autograd::Function<RopeFn> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k,
                               const Tensor &cos, const Tensor &sin, const OptTensor &wq,
                               const OptTensor &wk, double eps) {
    const c10::DeviceGuard guard(q.device());
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    int64_t q_st[4], k_st[4], qo_st[4], ko_st[4], cs[2];
    kernel_strides(q, q_st);
    kernel_strides(k, k_st);
    kernel_strides(qo, qo_st);
    kernel_strides(ko, ko_st);
    table_strides(cos, cs);
    check(fa_rope_qk_fwd(q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), cos.data_ptr(),
                         sin.data_ptr(), ptr_or_null(wq), ptr_or_null(wk), (float)eps,
                         (int)q.size(0), (int)q.size(1), (int)q.size(2), (int)k.size(2),
                         (int)q.size(3), q_st, k_st, qo_st, ko_st, cs, dtype_of(q), stream_of(q)),
          "fa_rope_qk_fwd");
    // the forward's inputs are needed again only to recompute a norm
    ctx->save_for_backward({wq ? q : Tensor(), wk ? k : Tensor(), cos, sin, wq.value_or(Tensor()),
                            wk.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    return {qo, ko};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const double eps = ctx->saved_data["eps"].toDouble();
    // the engine hands the gradients over in the outputs' shapes and dtype
    const auto dtype = grads[0].scalar_type();
    const at::Device device = grads[0].device();
    const c10::DeviceGuard guard(device);
    const int B = (int)grads[0].size(0), S = (int)grads[0].size(1), H = (int)grads[0].size(2),
              Hk = (int)grads[1].size(2), D = (int)grads[0].size(3);
    const bool norm[2] = {s[4].defined(), s[5].defined()};
    Tensor cos = s[2], sin = s[3], w[2];
    const bool one = cos.dim() == 3 && cos.size(0) == 1;
    check_saved(cos, cos.dim() == 2 ? at::DimVector{S, D} : at::DimVector{one ? 1 : B, S, D}, dtype,
                device);
    check_saved(sin, cos.sizes(), dtype, device);
    int64_t g_st[2][4], x_st[2][4], d_st[2][4], cs[2], sn[2];
    if (!table_ready(cos, cs) || !table_ready(sin, sn) || cs[0] != sn[0] || cs[1] != sn[1]) {
      cos = cos.clone(at::MemoryFormat::Contiguous);
      sin = sin.clone(at::MemoryFormat::Contiguous);
      table_ready(cos, cs);
    }
    const auto opt = cos.options();
    Tensor g[2], x[2], d[2], dw[2];
    for (int i = 0; i < 2; ++i) {
      g[i] = kernel_ready(grads[i].scalar_type() == dtype ? grads[i] : grads[i].to(dtype),
                          g_st[i]);
      if (norm[i]) {
        check_saved(s[i], g[i].sizes(), dtype, device);
        check_saved(s[4 + i], {D}, dtype, device);
        x[i] = kernel_ready(s[i], x_st[i]);
        w[i] = s[4 + i].is_contiguous() && aligned(s[4 + i])
                   ? s[4 + i] : s[4 + i].clone(at::MemoryFormat::Contiguous);
        dw[i] = at::empty({D}, opt);   // the weight's dtype
      } else {
        x[i] = g[i];   // read for a normed side only
        std::copy(g_st[i], g_st[i] + 4, x_st[i]);
      }
      d[i] = at::empty(g[i].sizes(), opt);
      kernel_strides(d[i], d_st[i]);
    }
    Tensor ws;
    if (norm[0] || norm[1])
      ws = at::empty({(int64_t)fa_rope_qk_workspace_bytes(B, S, H, Hk, D)}, opt.dtype(at::kByte));
    auto ptr = [](const Tensor &t) -> void * { return t.defined() ? t.data_ptr() : nullptr; };
    check(fa_rope_qk_bwd(g[0].data_ptr(), g[1].data_ptr(), x[0].data_ptr(), x[1].data_ptr(),
                         cos.data_ptr(), sin.data_ptr(), ptr(w[0]), ptr(w[1]), (float)eps,
                         d[0].data_ptr(), d[1].data_ptr(), static_cast<float *>(ptr(dw[0])),   // FA_DW_16
                         static_cast<float *>(ptr(dw[1])), ptr(ws),
                         ws.defined() ? (size_t)ws.numel() : 0, B, S, H, Hk, D, g_st[0], g_st[1],
                         x_st[0], x_st[1], d_st[0], d_st[1], cs, dtype_of(cos) | FA_DW_16,
                         stream_of(cos)),
          "fa_rope_qk_bwd");
    return {d[0], d[1], Tensor(), Tensor(), dw[0], dw[1], Tensor()};
  }
};

// (q_out, k_out) with the node recorded, or None for anything the kernels do
// not take in place as it is (other dtypes, devices and layouts, empty or
// misaligned tensors, tables that need a cast or have unequal strides or
// gradients, invalid arguments): the caller's general path copies, casts or
// raises.
std::optional<std::tuple<Tensor, Tensor>> rope(const Tensor &q, const Tensor &k, const Tensor &cos,
                                               const Tensor &sin, const OptTensor &wq,
                                               const OptTensor &wk, double eps) {
  if (q.dim() != 4 || k.dim() != 4 || !q.is_cuda()) return std::nullopt;
  const auto dt = q.scalar_type();
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), D = q.size(3), Hk = k.size(2);
  if ((dt != at::kHalf && dt != at::kBFloat16) || q.numel() == 0 || k.numel() == 0 ||
      (D != 16 && D != 32 && D != 64 && D != 128) || k.size(0) != B || k.size(1) != S ||
      k.size(3) != D || B > INT32_MAX || S > INT32_MAX ||
      (double)B * S * (double)std::max(H, Hk) > 2147483647.0)
    return std::nullopt;
  auto same = [&](const Tensor &t) {
    return t.scalar_type() == dt && t.device() == q.device() && aligned(t);
  };
  int64_t st[4];
  if (!same(q) || !same(k) || !kernel_strides(q, st) || !kernel_strides(k, st))
    return std::nullopt;
  int64_t c_st[2], s_st[2];
  for (const Tensor *t : {&cos, &sin}) {
    const int64_t d = t->dim();
    if ((d != 2 && d != 3) || t->size(d - 1) != D || t->size(d - 2) != S ||
        (d == 3 && t->size(0) != 1 && t->size(0) != B) || !same(*t) || t->requires_grad() ||
        !table_ready(*t, t == &cos ? c_st : s_st))
      return std::nullopt;
  }
  if (cos.sizes() != sin.sizes() || c_st[0] != s_st[0] || c_st[1] != s_st[1]) return std::nullopt;
  for (const OptTensor *w : {&wq, &wk}) {
    if (!*w) continue;
    if ((*w)->dim() != 1 || (*w)->size(0) != D || !same(**w) || !(*w)->is_contiguous() ||
        !(std::isfinite(eps) && eps >= 0.0))
      return std::nullopt;
  }
  variable_list r = RopeFn::apply(q, k, cos, sin, wq, wk, eps);
  return std::make_tuple(r[0], r[1]);
}

// The rotation by positions (rotary.py's apply_rotary_positions) and, with
// FA_ROTARY_INVERSE, its gradient: each is the other's.
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list rotate(const Tensor &q, const OptTensor &k, const Tensor &positions,
                              const Tensor &steps, double factor, int64_t dim, int64_t flags) {
    const c10::DeviceGuard guard(q.device());
    const bool two = k && k->defined();
    int64_t st[4][4] = {}, ps[2] = {positions.size(0) == 1 ? 0 : positions.stride(0),
                                    positions.stride(1)};
    const Tensor x = kernel_ready(q, st[0]);
    Tensor y = two ? kernel_ready(*k, st[1]) : Tensor();
    variable_list out = {at::empty(q.sizes(), q.options())};
    kernel_strides(out[0], st[2]);
    if (two) {
      out.push_back(at::empty(k->sizes(), k->options()));
      kernel_strides(out[1], st[3]);
    }
    if (positions.scalar_type() == at::kLong) flags |= FA_ROTARY_POS64;
    check(fa_rotary(x.data_ptr(), two ? y.data_ptr() : nullptr, out[0].data_ptr(),
                    two ? out[1].data_ptr() : nullptr, steps.data_ptr<int64_t>(), factor, (int)dim,
                    (int)flags, positions.data_ptr(), ps, (int)q.size(0), (int)q.size(1),
                    (int)q.size(2), two ? (int)k->size(2) : 0, (int)q.size(3), st[0], st[1], st[2],
                    st[3], dtype_of(q), stream_of(q)),
          "fa_rotary");
    return out;
  }

  static variable_list forward(AutogradContext *ctx, const Tensor &q, const OptTensor &k,
                               const Tensor &positions, const Tensor &steps, double factor,
                               int64_t dim, int64_t flags) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, steps});
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["dim"] = dim;
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["rows"] = positions.size(0);
    ctx->saved_data["wide"] = positions.scalar_type() == at::kLong;
    return rotate(q, k, positions, steps, factor, dim, flags);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t dim = ctx->saved_data["dim"].toInt();
    const int64_t flags = ctx->saved_data["flags"].toInt() ^ FA_ROTARY_INVERSE;
    const double factor = ctx->saved_data["factor"].toDouble();
    variable_list g, d(7);
    int side[2];
    for (size_t i = 0; i < grads.size(); ++i)   // a side that needs no gradient is not rotated
      if (grads[i].defined() && ctx->needs_input_grad(i)) {
        side[g.size()] = (int)i;
        g.push_back(grads[i]);
      }
    if (g.empty()) return d;
    check_saved(s[0], {ctx->saved_data["rows"].toInt(), g[0].size(1)},
                ctx->saved_data["wide"].toBool() ? at::kLong : at::kInt, g[0].device());
    check_saved(s[1], {dim / 2}, at::kLong, g[0].device());
    const Tensor steps = s[1].contiguous();
    const OptTensor second = g.size() > 1 ? OptTensor(g[1]) : OptTensor();
    const variable_list r =
        at::GradMode::is_enabled()
            ? RotaryFn::apply(g[0], second, s[0], steps, factor, dim, flags)
            : rotate(g[0], second, s[0], steps, factor, dim, flags);
    for (size_t i = 0; i < g.size(); ++i) d[side[i]] = r[i];
    return d;
  }
};

// Whether leaf `t` has a gradient accumulator that was made on another stream
// than the current one: an autograd graph of it lives there.  The engine makes
// that stream wait for a backward pass that reaches the leaf, which draws it
// into the capture of a pass that is being captured, and ending a capture with
// a stream not joined again ends the process.
bool held_on_another_stream(const Tensor &t) {
  if (!t.requires_grad() || !t.is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return false;
  const auto made = node->stream();
  return made && *made != c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device());
}

// (q_out, k_out or None) with the node recorded where a gradient is wanted, or
// None for anything the kernel does not take in place as it is (other dtypes,
// devices and layouts, empty or misaligned tensors, invalid arguments) and for
// a capture beside another graph of a leaf: rotary.py's general path copies or
// raises.  (The host time of a call is most of a decode step's: 13.9 us with the
// checks in Python.)
std::optional<std::tuple<Tensor, OptTensor>> rotary(const Tensor &q, const OptTensor &k,
                                                    const Tensor &positions, const Tensor &steps,
                                                    double factor, int64_t dim, int64_t flags) {
  if (q.dim() != 4 || !q.is_cuda() || q.numel() == 0) return std::nullopt;
  const auto dt = q.scalar_type();
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  int64_t st[4];
  if ((dt != at::kHalf && dt != at::kBFloat16) || D % 8 != 0 || D > 256 || dim > D ||
      !kernel_strides(q, st) || !aligned(q) || B > INT32_MAX || S > INT32_MAX)
    return std::nullopt;
  const bool two = k.has_value();
  if (two && (k->dim() != 4 || k->numel() == 0 || k->scalar_type() != dt ||
              k->device() != q.device() || k->size(0) != B || k->size(1) != S ||
              k->size(3) != D || !kernel_strides(*k, st) || !aligned(*k)))
    return std::nullopt;
  const auto pt = positions.scalar_type();
  if ((pt != at::kInt && pt != at::kLong) || positions.device() != q.device() ||
      steps.device() != q.device())
    return std::nullopt;
  if (positions.dim() < 1 || positions.dim() > 2) return std::nullopt;
  const Tensor p = positions.dim() == 1 ? positions.unsqueeze(0) : positions;
  if (p.size(1) != S || (p.size(0) != 1 && p.size(0) != B)) return std::nullopt;
  variable_list r;
  if (at::GradMode::is_enabled() && (q.requires_grad() || (two && k->requires_grad()))) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None &&
        (held_on_another_stream(q) || (two && held_on_another_stream(*k))))
      return std::nullopt;
    r = RotaryFn::apply(q, k, p, steps, factor, dim, flags);
  } else {
    r = RotaryFn::rotate(q, k, p, steps, factor, dim, flags);
  }
  return std::make_tuple(r[0], two ? OptTensor(r[1]) : OptTensor());
}

// The paged cache's calls (paged.py), for arguments that the kernels take in
// place as they are; None for any others.  `cache` is the address of the
// fa_paged_cache of the table's width, `like` one of the cache's tensors.
struct PagedCall {
  const fa_paged_cache *cache;
  const Tensor &like;
  at::ScalarType dtype;
  int64_t D, B = 0;
  int code() const { return dtype == at::kHalf ? FA_DTYPE_F16 : FA_DTYPE_BF16; }
  bool rows(const Tensor &t, int64_t (&st)[4]) const {
    return t.dim() == 4 && t.scalar_type() == dtype && t.device() == like.device() &&
           t.numel() != 0 && t.size(3) == D && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX &&
           kernel_strides(t, st) && aligned(t);
  }
  bool counts(const Tensor &t) const {
    return t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kInt &&
           t.device() == like.device() && (B == 1 || t.stride(0) == 1);
  }
  bool table(const Tensor &t) const {
    return t.dim() == 2 && t.size(0) == B && t.size(1) == cache->width &&
           t.scalar_type() == at::kInt && t.device() == like.device() && t.stride(0) >= 0 &&
           (t.stride(1) == 1 || t.size(1) == 1);
  }
};

const int32_t *ints(const OptTensor &t) { return t ? t->data_ptr<int32_t>() : nullptr; }

// (done, q_out or None)
std::tuple<bool, OptTensor> paged_append(int64_t cache, const Tensor &like, bool half, int64_t D,
                                         const Tensor &table, const Tensor &k, const Tensor &v,
                                         const OptTensor &q, const Tensor &start,
                                         const OptTensor &counts, const OptTensor &steps,
                                         double factor, int64_t dim, int64_t flags) {
  PagedCall c{reinterpret_cast<const fa_paged_cache *>(cache), like,
              half ? at::kHalf : at::kBFloat16, D};
  int64_t k_st[4], v_st[4], q_st[4] = {}, qo_st[4] = {};
  const std::tuple<bool, OptTensor> no{false, OptTensor()};
  if (!like.is_cuda() || !c.rows(k, k_st) || !c.rows(v, v_st) || k.sizes() != v.sizes() ||
      k.size(2) != c.cache->heads)
    return no;
  const int64_t S = k.size(1);
  c.B = k.size(0);
  if (!c.table(table) || !c.counts(start) || (counts && !c.counts(*counts)) ||
      (steps && (steps->device() != like.device() || dim > D)))
    return no;
  if (q && (!c.rows(*q, q_st) || q->size(0) != c.B || q->size(1) != S)) return no;
  const c10::DeviceGuard guard(like.device());
  Tensor out;
  if (q) {
    out = at::empty(q->sizes(), q->options());
    kernel_strides(out, qo_st);
  }
  check(fa_paged_append(c.cache, table.data_ptr<int32_t>(), table.stride(0), k.data_ptr(),
                        v.data_ptr(), q ? q->data_ptr() : nullptr, q ? out.data_ptr() : nullptr,
                        ints(OptTensor(start)), ints(counts),
                        steps ? steps->data_ptr<int64_t>() : nullptr, factor, (int)dim, (int)flags,
                        (int)c.B, (int)S, q ? (int)q->size(2) : 0, (int)D, k_st, v_st, q_st, qo_st,
                        c.code(), stream_of(like)),
        "fa_paged_append");
  return {true, q ? OptTensor(out) : OptTensor()};
}

std::optional<std::tuple<Tensor, Tensor>> paged_read(int64_t cache, const Tensor &like, bool half,
                                                     int64_t D, const Tensor &table,
                                                     const Tensor &start, int64_t n,
                                                     const OptTensor &counts) {
  PagedCall c{reinterpret_cast<const fa_paged_cache *>(cache), like,
              half ? at::kHalf : at::kBFloat16, D};
  c.B = table.dim() == 2 ? table.size(0) : 0;
  if (!like.is_cuda() || c.B <= 0 || n <= 0 || n > INT32_MAX || !c.table(table) ||
      !c.counts(start) || (counts && !c.counts(*counts)))
    return std::nullopt;
  const c10::DeviceGuard guard(like.device());
  const auto opt = like.options().dtype(c.dtype);
  Tensor k = at::empty({c.B, n, c.cache->heads, D}, opt), v = at::empty(k.sizes(), opt);
  check(fa_paged_read(c.cache, table.data_ptr<int32_t>(), table.stride(0), k.data_ptr(),
                      v.data_ptr(), ints(OptTensor(start)), ints(counts), (int)c.B, (int)n, (int)D,
                      c.code(), stream_of(like)),
        "fa_paged_read");
  return std::make_tuple(k, v);
}

std::optional<std::tuple<Tensor, OptTensor>> paged_attend(int64_t cache, const Tensor &like,
                                                          bool half, int64_t D, const Tensor &q,
                                                          const Tensor &table,
                                                          const Tensor &lengths,
                                                          const OptTensor &counts, double scale,
                                                          bool want_lse) {
  PagedCall c{reinterpret_cast<const fa_paged_cache *>(cache), like,
              half ? at::kHalf : at::kBFloat16, D};
  int64_t q_st[4];
  if (!like.is_cuda() || !c.rows(q, q_st)) return std::nullopt;
  const int64_t Sq = q.size(1), H = q.size(2), Hk = c.cache->heads;
  c.B = q.size(0);
  if (H > INT32_MAX || H % Hk != 0 || !c.table(table) || !c.counts(lengths) ||
      (counts && !c.counts(*counts)))
    return std::nullopt;
  const c10::DeviceGuard guard(like.device());
  Tensor out = at::empty(q.sizes(), q.options()), lse, ws;
  if (want_lse) lse = at::empty({c.B, H, Sq}, q.options().dtype(at::kFloat));
  // (its memory is the allocator's again on return, for later work of this stream)
  const size_t nb = fa_paged_attn_workspace_bytes((int)c.B, (int)Sq, (int)H, (int)Hk, (int)D);
  if (nb) ws = at::empty({(int64_t)nb}, q.options().dtype(at::kByte));
  check(fa_paged_attn(q.data_ptr(), c.cache, table.data_ptr<int32_t>(), table.stride(0),
                      lengths.data_ptr<int32_t>(), ints(counts), out.data_ptr(),
                      want_lse ? lse.data_ptr<float>() : nullptr, nb ? ws.data_ptr() : nullptr, nb,
                      (int)c.B, (int)Sq, (int)H, (int)D, q_st, (float)scale, c.code(),
                      stream_of(like)),
        "fa_paged_attn");
  return std::make_tuple(out, want_lse ? OptTensor(lse) : OptTensor());
}

}  // namespace

PYBIND11_MODULE(_fa_torch, m) {
  // This module calls the library's entry points with the argument lists of
  // the header it was compiled against; a library built from another ABI
  // version (the two .so files are built separately) would take them
  // without an error.  Refuse to load then: the Python autograd path, which
  // checks the version itself, takes over.
  if (fa_abi_version() != FA_ABI_VERSION) {
    PyErr_Format(PyExc_ImportError,
                 "_fa_torch was built for libfa_mi355x ABI %d, the loaded library has ABI %d: "
                 "rebuild both (flash_attn_volta.build)",
                 (int)FA_ABI_VERSION, (int)fa_abi_version());
    throw pybind11::error_already_set();
  }
  m.doc() = "C++ autograd nodes of flash_attn_volta's flash_attn / flash_attn_gqa / apply_rotary_qk / "
            "apply_rotary_positions";
  m.def("make_plan", &make_plan, "register a launch plan (ints, sm_scale) -> handle");
  m.def("rope", &rope, "QK-norm + rotary prologue, recording the C++ backward node, or None");
  m.def("rotary", &rotary, "rotation by positions, recording the C++ backward node, or None");
  m.def("paged_append", &paged_append, "append_paged -> (done, q_out or None)");
  m.def("paged_read", &paged_read, "read_paged -> (k, v), or None");
  m.def("paged_attend", &paged_attend, "attend_paged -> (out, lse or None), or None");
  m.def("held_on_another_stream", &held_on_another_stream,
        "a leaf's gradient accumulator was made on another stream");
  m.def("attn", &attn, "forward of a plan, recording the C++ backward node");
  m.attr("PLAN_INTS") = (int64_t)kPlanInts;
}
