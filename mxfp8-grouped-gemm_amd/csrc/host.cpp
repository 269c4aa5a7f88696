// Native host path of the Python entry points: checks, output allocation and
// the library call in one step.
//
// A small call (a few hundred tokens, small layers) is bound by the host: in
// Python an op spends 20 to 60 us on attribute reads, allocations and a ctypes
// call of 20 to 30 arguments, for kernels of 3 to 20 us.  Each function below
// takes the plain case of its op (device tensors of the right type, laid out as
// the kernels read them).  For anything else it returns None and touches
// nothing: the caller then runs the Python form, which converts, splits or
// raises.  A result is a tensor or a tuple; an int is a library status.
// Like torch's own ops, the functions run without the GIL (an allocation or a
// launch on a full queue can block) and raise torch's exceptions (a trainer
// catches torch.OutOfMemoryError).
//
// Library functions are reached through addresses handed in once by bind(), so
// this module does not link against libmxgg.so; bind() refuses a library of
// another ABI version than the header this module was compiled with.
#include <torch/extension.h>

#include <cstring>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <variant>
#include <vector>

#include "../../include/mxgg.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Lib {
#define MXGG_FN(name) decltype(&::mxgg_##name) name = nullptr;
#define MXGG_FNS                                                                            \
  MXGG_FN(quant_dim0) MXGG_FN(quant_dim1) MXGG_FN(quant_dual) MXGG_FN(zero_rows_past_groups) \
  MXGG_FN(grouped_fwd) MXGG_FN(grouped_fwd_split) MXGG_FN(grouped_fwd_swiglu_quant)          \
  MXGG_FN(grouped_fwd_swiglu_quant_keep_h) MXGG_FN(grouped_wgrad) MXGG_FN(swiglu_bwd_quant)  \
  MXGG_FN(gather_quant_dual) MXGG_FN(gather_quant_dim0) MXGG_FN(combine)                     \
  MXGG_FN(route_topk) MXGG_FN(route_topk_grad) MXGG_FN(norm) MXGG_FN(norm_grad)              \
  MXGG_FN(norm_grad_workspace_bytes) MXGG_FN(adamw_step) MXGG_FN(last_error)                 \
  MXGG_FN(linear_cross_entropy) MXGG_FN(linear_cross_entropy_workspace_bytes)                \
  MXGG_FN(linear_cross_entropy_grad) MXGG_FN(linear_cross_entropy_grad_workspace_bytes)
  MXGG_FNS
#undef MXGG_FN
};
Lib lib;

void bind(const py::dict& address) {
  const auto version = reinterpret_cast<decltype(&::mxgg_abi_version)>(
      address["mxgg_abi_version"].cast<uintptr_t>())();
  if (version != MXGG_ABI_VERSION)
    throw std::runtime_error("built for ABI version " + std::to_string(MXGG_ABI_VERSION) +
                             ", the library has " + std::to_string(version));
  Lib l;
#define MXGG_FN(name) \
  l.name = reinterpret_cast<decltype(l.name)>(address["mxgg_" #name].cast<uintptr_t>());
  MXGG_FNS
#undef MXGG_FN
  lib = l;
}

constexpr int64_t kMaxOperandBytes = 0x7FFFFFF0;  // the C ABI's bound on (rows - 1) * ld + K

// A device tensor with memory of its own behind it (no fake, batched or
// otherwise wrapped tensor).
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == c10::kStrided && t.has_storage() &&
         !t.key_set().has(c10::DispatchKey::Python) && t.numel() > 0 &&
         t.const_data_ptr() != nullptr;
}
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// 2-D bf16 rows the kernels read in place.
bool bf16_rows(const Tensor& t) {
  return plain(t) && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 &&
         t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned(t.const_data_ptr(), 16);
}
bool bytes(const Tensor& t) {
  const auto d = t.scalar_type();
  return plain(t) && (d == at::kFloat8_e4m3fn || d == at::kByte);
}
// Group ends used as they are.
bool ends_ok(const OptTensor& e, const Tensor& like) {
  return !e || (plain(*e) && e->scalar_type() == at::kInt && e->dim() == 1 &&
                e->is_contiguous() && e->device() == like.device());
}
const int32_t* ends_ptr(const OptTensor& e) { return e ? e->const_data_ptr<int32_t>() : nullptr; }

int64_t ld16(int64_t n) { return std::max<int64_t>(16, (n + 15) / 16 * 16); }
int64_t padded_capacity(int64_t tokens, int64_t groups) {
  return groups == 0 ? (tokens + 31) / 32 * 32 : (tokens + 31 * groups + 127) / 128 * 128;
}
Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type).requires_grad(false));
}
// Storage of block-major scales, [nblk][round_up(rows, 16)], and the logical
// [rows, nblk] view of it.
Tensor block_major(int64_t rows, int64_t nblk, const Tensor& like) {
  return empty({nblk, ld16(rows)}, like, at::kByte);
}
Tensor rows_view(const Tensor& buf, int64_t rows) {
  return buf.as_strided({rows, buf.size(0)}, {1, buf.stride(0)});
}
void* vp(const Tensor& t) { return t.data_ptr(); }
const void* cp(const Tensor& t) { return t.const_data_ptr(); }
void* st(int64_t stream) { return reinterpret_cast<void*>(stream); }

using Result = std::variant<std::monostate, int, Tensor, std::tuple<Tensor, Tensor>,
                            std::tuple<Tensor, Tensor, Tensor>,
                            std::tuple<Tensor, Tensor, OptTensor>,
                            std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>,
                            std::tuple<Tensor, Tensor, Tensor, Tensor, OptTensor>,
                            std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, OptTensor>>;
Result none() { return std::monostate{}; }

// E8M0 scales [rows, nblk] (or [E, rows, nblk]) stored block-major, as the
// library's casts return them; the conditions are the Python form's.
int64_t readable(const Tensor& t) {
  return (int64_t)t.storage().nbytes() - t.storage_offset() * t.element_size();
}
bool scale_bytes(const Tensor& s, const Tensor& of) {
  const auto d = s.scalar_type();
  return plain(s) && s.device() == of.device() &&
         (d == at::kByte || d == at::kFloat8_e8m0fnu || d == at::kFloat8_e4m3fn || d == at::kChar);
}
bool scales_2d(const Tensor& s, const Tensor& of, int64_t rows, int64_t nblk) {
  return scale_bytes(s, of) && s.dim() == 2 && s.size(0) == rows &&
         s.size(1) == nblk && (s.stride(0) == 1 || rows == 1) && s.stride(1) >= rows &&
         s.stride(1) % 4 == 0 && aligned(cp(s), 4) &&
         readable(s) >= (nblk - 1) * s.stride(1) + (rows + 3) / 4 * 4;
}
bool scales_3d(const Tensor& s, const Tensor& of, int64_t E, int64_t rows, int64_t nblk) {
  return scale_bytes(s, of) && s.dim() == 3 && s.size(0) == E &&
         s.size(1) == rows && s.size(2) == nblk && (s.stride(1) == 1 || rows == 1) &&
         s.stride(2) % 4 == 0 && (E == 1 || s.stride(0) % 4 == 0) && aligned(cp(s), 4) &&
         s.stride(2) >= rows && (E == 1 || s.stride(0) >= rows) &&
         readable(s) >= (E - 1) * s.stride(0) + (nblk - 1) * s.stride(2) + (rows + 3) / 4 * 4;
}

Result dim0(const Tensor& x, bool block, int mode, int64_t stream) {
  if (!plain(x) || x.scalar_type() != at::kBFloat16 || x.dim() < 1 || !x.is_contiguous() ||
      x.size(-1) % 32 != 0 || !aligned(cp(x), 16))
    return none();
  const int64_t K = x.size(-1), rows = x.numel() / K, nblk = K / 32;
  Tensor q = empty(x.sizes(), x, at::kFloat8_e4m3fn);
  auto size = x.sizes().vec();
  size.back() = nblk;
  Tensor s;
  int64_t lds;
  if (block) {
    lds = ld16(rows);
    Tensor buf = block_major(rows, nblk, x);
    std::vector<int64_t> stride(size.size());
    int64_t acc = 1;
    for (size_t d = size.size() - 1; d-- > 0;) {
      stride[d] = acc;
      acc *= size[d];
    }
    stride.back() = lds;
    s = buf.as_strided(size, stride);
  } else {
    lds = nblk;
    s = empty(size, x, at::kByte);
  }
  const int rc = lib.quant_dim0(cp(x), rows, K, K, vp(q), K, vp(s), lds,
                                block ? MXGG_SCALES_BLOCK_MAJOR : MXGG_SCALES_ROW_MAJOR, mode,
                                st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(q, s);
}

// cap: columns of the token-axis cast, 0 = padded_capacity.
Result dim1(const Tensor& x, const OptTensor& ends, bool block, int64_t cap, int mode,
                int64_t stream) {
  if (!bf16_rows(x) || x.size(1) % 8 != 0 || !ends_ok(ends, x)) return none();
  const int64_t M = x.size(0), C = x.size(1), E = ends ? ends->numel() : 0;
  if (cap == 0) cap = padded_capacity(M, E);
  Tensor qt = empty({C, cap}, x, at::kFloat8_e4m3fn);
  Tensor buf = block ? block_major(C, cap / 32, x) : empty({C, cap / 32}, x, at::kByte);
  OptTensor pad;
  if (ends) pad = empty({E}, x, at::kInt);
  const int rc = lib.quant_dim1(
      cp(x), M, C, x.stride(0), ends_ptr(ends), E, cap, vp(qt), cap, vp(buf), buf.stride(0),
      block ? MXGG_SCALES_BLOCK_MAJOR : MXGG_SCALES_ROW_MAJOR,
      pad ? pad->data_ptr<int32_t>() : nullptr, mode, st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(qt, block ? rows_view(buf, C) : buf, pad);
}

Result dual(const Tensor& x, const OptTensor& ends, int64_t cap, int mode, int64_t stream) {
  if (!bf16_rows(x) || x.size(1) % 32 != 0 || !ends_ok(ends, x)) return none();
  const int64_t M = x.size(0), C = x.size(1), E = ends ? ends->numel() : 0;
  if (cap == 0) cap = padded_capacity(M, E);
  Tensor q = empty({M, C}, x, at::kFloat8_e4m3fn), qt = empty({C, cap}, x, at::kFloat8_e4m3fn);
  Tensor sb = block_major(M, C / 32, x), stb = block_major(C, cap / 32, x);
  OptTensor pad;
  if (ends) pad = empty({E}, x, at::kInt);
  const int rc = lib.quant_dual(cp(x), M, C, x.stride(0), ends_ptr(ends), E, cap, vp(q), C, vp(sb),
                                sb.stride(0), vp(qt), cap, vp(stb), stb.stride(0),
                                MXGG_SCALES_BLOCK_MAJOR, pad ? pad->data_ptr<int32_t>() : nullptr,
                                mode, st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(q, rows_view(sb, M), qt, rows_view(stb, C), pad);
}

// Operands of the grouped forward, checked.
struct FwdIn {
  int64_t M, K, E, N;
  const void *as = nullptr, *ws = nullptr;
  int64_t ldas = 0, wsg = 0, ldws = 0;
};
bool fwd_in(const Tensor& a, const Tensor& w, const OptTensor& ends, const OptTensor& as,
            const OptTensor& ws, FwdIn& in) {
  if (!bytes(a) || !bytes(w) || a.dim() != 2 || w.dim() != 3 || a.stride(1) != 1 ||
      w.stride(2) != 1 || a.size(1) != w.size(2) || a.device() != w.device() ||
      as.has_value() != ws.has_value() || !ends_ok(ends, a))
    return false;
  in.M = a.size(0);
  in.K = a.size(1);
  in.E = w.size(0);
  in.N = w.size(1);
  if (in.K % 32 != 0 || (ends ? ends->numel() != in.E : in.E != 1) ||
      (in.M - 1) * a.stride(0) + in.K > kMaxOperandBytes)
    return false;
  if (as) {
    if (!scales_2d(*as, a, in.M, in.K / 32) || !scales_3d(*ws, a, in.E, in.N, in.K / 32)) return false;
    in.as = cp(*as);
    in.ldas = as->stride(1);
    in.ws = cp(*ws);
    in.wsg = ws->stride(0);
    in.ldws = ws->stride(2);
  }
  return true;
}

// split: workspace bytes of the split entry, 0 for the unsplit one.
Result mm(const Tensor& a, const Tensor& w, const OptTensor& ends, const OptTensor& as,
              const OptTensor& ws, bool f32, int64_t split, int64_t stream) {
  FwdIn in;
  if (!fwd_in(a, w, ends, as, ws, in) || in.N % 4 != 0) return none();
  Tensor out = empty({in.M, in.N}, a, f32 ? at::kFloat : at::kBFloat16);
  const int type = f32 ? MXGG_OUT_F32 : MXGG_OUT_BF16;
  int rc;
  if (split > 0) {
    Tensor scratch = empty({split}, a, at::kByte);
    rc = lib.grouped_fwd_split(cp(a), a.stride(0), in.as, in.ldas, cp(w), w.stride(0), w.stride(1),
                               in.ws, in.wsg, in.ldws, ends_ptr(ends), in.E, in.M, in.N, in.K,
                               vp(out), in.N, type, vp(scratch), split, st(stream));
  } else {
    rc = lib.grouped_fwd(cp(a), a.stride(0), in.as, in.ldas, cp(w), w.stride(0), w.stride(1),
                         in.ws, in.wsg, in.ldws, ends_ptr(ends), in.E, in.M, in.N, in.K, vp(out),
                         in.N, type, st(stream));
  }
  if (rc != MXGG_OK) return rc;
  return out;
}

Result mm_swiglu(const Tensor& a, const Tensor& w, const OptTensor& ends, const OptTensor& as,
                     const OptTensor& ws, int mode, bool keep, int64_t stream) {
  FwdIn in;
  if (!fwd_in(a, w, ends, as, ws, in) || in.N % 256 != 0) return none();
  const int64_t F = in.N / 2;
  Tensor q = empty({in.M, F}, a, at::kFloat8_e4m3fn), buf = block_major(in.M, F / 32, a);
  Tensor h;
  int rc;
  if (keep) {
    h = empty({in.M, in.N}, a, at::kBFloat16);
    rc = lib.grouped_fwd_swiglu_quant_keep_h(
        cp(a), a.stride(0), in.as, in.ldas, cp(w), w.stride(0), w.stride(1), in.ws, in.wsg,
        in.ldws, ends_ptr(ends), in.E, in.M, F, in.K, vp(h), in.N, vp(q), F, vp(buf),
        buf.stride(0), MXGG_SCALES_BLOCK_MAJOR, mode, st(stream));
    // the kernel writes no row past the last group end
    if (rc == MXGG_OK && ends)
      rc = lib.zero_rows_past_groups(vp(h), in.M, 2 * in.N, 2 * in.N, ends_ptr(ends), in.E,
                                     st(stream));
  } else {
    rc = lib.grouped_fwd_swiglu_quant(
        cp(a), a.stride(0), in.as, in.ldas, cp(w), w.stride(0), w.stride(1), in.ws, in.wsg,
        in.ldws, ends_ptr(ends), in.E, in.M, F, in.K, vp(q), F, vp(buf), buf.stride(0),
        MXGG_SCALES_BLOCK_MAJOR, mode, st(stream));
  }
  if (rc != MXGG_OK) return rc;
  if (keep) return std::make_tuple(q, rows_view(buf, in.M), h);
  return std::make_tuple(q, rows_view(buf, in.M));
}

// Unsplit weight gradient into a new dW.
Result wgrad(const Tensor& go, const Tensor& ia, const Tensor& ends, const OptTensor& gs,
                 const OptTensor& is, bool f32, int64_t stream) {
  if (!bytes(go) || !bytes(ia) || go.dim() != 2 || ia.dim() != 2 || go.stride(1) != 1 ||
      ia.stride(1) != 1 || go.size(1) != ia.size(1) || go.device() != ia.device() ||
      gs.has_value() != is.has_value() || !ends_ok(ends, go))
    return none();
  const int64_t N = go.size(0), K = ia.size(0), M = go.size(1), E = ends.numel();
  if (K % 4 != 0 || M % 32 != 0 || (N - 1) * go.stride(0) + M > kMaxOperandBytes ||
      (K - 1) * ia.stride(0) + M > kMaxOperandBytes)
    return none();
  if (gs && (!scales_2d(*gs, go, N, M / 32) || !scales_2d(*is, go, K, M / 32))) return none();
  Tensor dw = empty({E, N, K}, go, f32 ? at::kFloat : at::kBFloat16);
  const int rc = lib.grouped_wgrad(
      cp(go), go.stride(0), gs ? cp(*gs) : nullptr, gs ? gs->stride(1) : 0, cp(ia), ia.stride(0),
      is ? cp(*is) : nullptr, is ? is->stride(1) : 0, ends.const_data_ptr<int32_t>(), E, M, N, K,
      vp(dw), f32 ? MXGG_OUT_F32 : MXGG_OUT_BF16, 0, st(stream));
  if (rc != MXGG_OK) return rc;
  return dw;
}

Result swiglu_bwd(const Tensor& h, const Tensor& da, const OptTensor& ends, int mode,
                      int64_t stream) {
  if (!bf16_rows(h) || !bf16_rows(da) || h.size(1) % 64 != 0 || da.size(0) != h.size(0) ||
      da.size(1) != h.size(1) / 2 || !ends_ok(ends, h) || h.device() != da.device())
    return none();
  const int64_t M = h.size(0), F = da.size(1), E = ends ? ends->numel() : 0;
  const int64_t cap = padded_capacity(M, E);
  const uint16_t* gate = static_cast<const uint16_t*>(cp(h));
  Tensor q = empty({M, 2 * F}, h, at::kFloat8_e4m3fn), sb = block_major(M, 2 * F / 32, h);
  Tensor qt = empty({2 * F, cap}, h, at::kFloat8_e4m3fn), stb = block_major(2 * F, cap / 32, h);
  Tensor at = empty({F, cap}, h, at::kFloat8_e4m3fn), atb = block_major(F, cap / 32, h);
  OptTensor pad;
  if (ends) pad = empty({E}, h, at::kInt);
  const int rc = lib.swiglu_bwd_quant(
      gate, gate + F, h.stride(0), cp(da), da.stride(0), M, F, ends_ptr(ends), E, cap, vp(q), 2 * F,
      vp(sb), sb.stride(0), vp(qt), cap, vp(stb), stb.stride(0), vp(at), cap, vp(atb),
      atb.stride(0), pad ? pad->data_ptr<int32_t>() : nullptr, nullptr, 2 * F,
      MXGG_SCALES_BLOCK_MAJOR, mode, st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(q, rows_view(sb, M), qt, rows_view(stb, 2 * F), at, rows_view(atb, F), pad);
}

Result zero_rows(const Tensor& out, const Tensor& ends, int64_t stream) {
  if (!plain(out) || out.dim() != 2 || out.stride(1) != 1 || !ends_ok(ends, out)) return none();
  const int64_t e = out.element_size();
  const int rc = lib.zero_rows_past_groups(vp(out), out.size(0), out.size(1) * e, out.stride(0) * e,
                                           ends.const_data_ptr<int32_t>(), ends.numel(),
                                           st(stream));
  return rc;
}

// Routing: src / perm / offs are a plan's tensors.
bool row_scores(const Tensor& s, const Tensor& of, int64_t slots) {
  return plain(s) && s.scalar_type() == at::kFloat && s.is_contiguous() && s.numel() == slots &&
         s.device() == of.device();
}
Result gather_dual(const Tensor& x, const Tensor& src, const Tensor& offs, int topk,
                       const OptTensor& scale, int mode, int64_t stream) {
  if (!bf16_rows(x) || x.size(1) % 32 != 0 || !ends_ok(src, x) || !ends_ok(offs, x) ||
      (scale && !row_scores(*scale, x, x.size(0) * topk)))
    return none();
  const int64_t M = src.numel(), C = x.size(1), E = offs.numel(), cap = padded_capacity(M, E);
  Tensor q = empty({M, C}, x, at::kFloat8_e4m3fn), qt = empty({C, cap}, x, at::kFloat8_e4m3fn);
  Tensor sb = block_major(M, C / 32, x), stb = block_major(C, cap / 32, x);
  Tensor pad = empty({E}, x, at::kInt);
  const int rc = lib.gather_quant_dual(
      cp(x), x.size(0), C, x.stride(0), src.const_data_ptr<int32_t>(), topk,
      scale ? scale->const_data_ptr<float>() : nullptr, M, offs.const_data_ptr<int32_t>(), E, cap,
      vp(q), C, vp(sb), sb.stride(0), vp(qt), cap, vp(stb), stb.stride(0),
      MXGG_SCALES_BLOCK_MAJOR, pad.data_ptr<int32_t>(), mode, st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(q, rows_view(sb, M), qt, rows_view(stb, C), pad);
}

Result gather_dim0(const Tensor& x, const Tensor& src, int topk, int mode, int64_t stream) {
  if (!bf16_rows(x) || x.size(1) % 32 != 0 || !ends_ok(src, x)) return none();
  const int64_t M = src.numel(), C = x.size(1);
  Tensor q = empty({M, C}, x, at::kFloat8_e4m3fn), sb = block_major(M, C / 32, x);
  const int rc = lib.gather_quant_dim0(cp(x), x.size(0), C, x.stride(0),
                                       src.const_data_ptr<int32_t>(), topk, M, vp(q), C, vp(sb),
                                       sb.stride(0), MXGG_SCALES_BLOCK_MAJOR, mode, st(stream));
  if (rc != MXGG_OK) return rc;
  return std::make_tuple(q, rows_view(sb, M));
}

Result combine(const Tensor& y, const Tensor& perm, int64_t tokens, int topk,
                   const OptTensor& scores, int64_t stream) {
  if (!bf16_rows(y) || y.size(1) % 8 != 0 || !ends_ok(perm, y) || perm.numel() != tokens * topk ||
      (scores && !row_scores(*scores, y, tokens * topk)))
    return none();
  Tensor out = empty({tokens, y.size(1)}, y, at::kBFloat16);
  const int rc = lib.combine(cp(y), y.size(0), y.size(1), y.stride(0),
                             perm.const_data_ptr<int32_t>(),
                             scores ? scores->const_data_ptr<float>() : nullptr, tokens, topk,
                             vp(out), out.stride(0), st(stream));
  if (rc != MXGG_OK) return rc;
  return out;
}

// The operators below are differentiable here as well: an autograd function in
// Python costs more host time than their kernels take on small inputs.  Their
// backward passes launch on the stream of the forward pass, where autograd runs
// them.  Arguments that the library would refuse are left to the Python form.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == MXGG_OK, what, ": status ", rc, ": ", lib.last_error());
}
// A plain struct kept for the backward pass.
template <class T>
void keep(AutogradContext* ctx, const char* name, const T& v) {
  ctx->saved_data[name] = std::string(reinterpret_cast<const char*>(&v), sizeof(T));
}
template <class T>
T kept(AutogradContext* ctx, const char* name) {
  T v;
  const std::string s = ctx->saved_data[name].toStringRef();
  std::memcpy(&v, s.data(), sizeof(T));
  return v;
}
bool grad_needed(const OptTensor& a) { return a && a->requires_grad(); }
bool f32_or_bf16(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
int32_t type_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? MXGG_OUT_BF16 : MXGG_OUT_F32;
}
// A tangent of forward-mode differentiation, which these operators do not propagate.
bool tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool tangent(const OptTensor& t) { return t && tangent(*t); }
void* vp_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const void* cp_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Refuses a backward pass under create_graph: the gradients would be constants in its
// graph, and second derivatives would leave their part out unnoticed.
void first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " cannot be differentiated twice (create_graph)");
}

// (expert_idx, weights) and, for the gradient, what it needs of the chosen.
variable_list route_forward(const Tensor& logits, const float* bias,
                            const mxgg_route_options& o, bool keep_selected, int64_t stream) {
  const int64_t tokens = logits.size(0);
  Tensor idx = empty({tokens, o.topk}, logits, at::kInt);
  Tensor weights = empty({tokens, o.topk}, logits, at::kFloat);
  Tensor selected;
  if (keep_selected) selected = empty({tokens, o.topk}, logits, at::kFloat);
  check(lib.route_topk(cp(logits), tokens, bias, &o,
                       idx.data_ptr<int32_t>(), weights.data_ptr<float>(),
                       static_cast<float*>(vp_or_null(selected)), st(stream)),
        "route_topk");
  return {idx, weights, selected};
}

struct RouteTopK : torch::autograd::Function<RouteTopK> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const float* bias,
                               const mxgg_route_options& o, int64_t stream) {
    variable_list r = route_forward(logits, bias, o, true, stream);
    const bool whole = o.score == MXGG_SCORE_SOFTMAX && !o.renormalize;
    ctx->save_for_backward({r[0], r[2], whole ? logits : Tensor()});
    keep(ctx, "options", o);
    ctx->saved_data["stream"] = stream;
    ctx->mark_non_differentiable({r[0]});
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order("route_topk");
    const variable_list saved = ctx->get_saved_variables();
    const auto o = kept<mxgg_route_options>(ctx, "options");
    const Tensor d = grads[1].to(at::kFloat).contiguous();
    Tensor out = empty({d.size(0), o.experts}, d,
                       o.dtype == MXGG_OUT_BF16 ? at::kBFloat16 : at::kFloat);
    check(lib.route_topk_grad(d.const_data_ptr<float>(), saved[0].const_data_ptr<int32_t>(),
                              saved[1].const_data_ptr<float>(), cp_or_null(saved[2]), d.size(0),
                              &o, vp(out), st(ctx->saved_data["stream"].toInt())),
          "route_topk_grad");
    return {out, Tensor(), Tensor(), Tensor()};
  }
};

Result route_topk(const Tensor& logits, const OptTensor& bias, int64_t topk, int64_t groups,
                  int64_t top_groups, int score, int group_best, bool renormalize, double scale,
                  int64_t stream) {
  if (!plain(logits) || tangent(logits) || logits.dim() != 2 || !f32_or_bf16(logits) || !logits.is_contiguous() ||
      (bias && (!plain(*bias) || bias->scalar_type() != at::kFloat || bias->dim() != 1 ||
                bias->size(0) != logits.size(1) || !bias->is_contiguous() ||
                bias->device() != logits.device())))
    return none();
  const int64_t E = logits.size(1);
  if (E > 1024 || topk < 1 || topk > std::min<int64_t>(E, 32) || groups < 1 || groups > 64 ||
      E % groups != 0 || top_groups < 1 || top_groups > groups ||
      (group_best != 1 && group_best != 2) || logits.size(0) >= INT64_C(1) << 24)
    return none();
  const mxgg_route_options o{E,          topk,           groups,     top_groups,
                             score,      type_of(logits), group_best, renormalize,
                             (float)scale};
  const float* b = bias ? bias->const_data_ptr<float>() : nullptr;
  variable_list r = at::GradMode::is_enabled() && logits.requires_grad()
                        ? RouteTopK::apply(logits, b, o, stream)
                        : route_forward(logits, b, o, false, stream);
  return std::make_tuple(r[0], r[1]);
}

// Rows that the norm kernels read in place: the row stride, or -1.
int64_t row_stride(const Tensor& t) {
  const int64_t cols = t.size(-1);
  if (t.is_contiguous()) return cols;
  return t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= cols ? t.stride(0) : -1;
}
variable_list norm_forward(const Tensor& x, const OptTensor& w, const OptTensor& b,
                           const mxgg_norm_options& o, bool keep_stats, int64_t stream) {
  Tensor y = empty(x.sizes(), x, x.scalar_type()), stats;
  if (keep_stats) stats = empty({2, o.rows}, x, at::kFloat);
  check(lib.norm(cp(x), row_stride(x), w ? cp(*w) : nullptr, b ? cp(*b) : nullptr, &o, vp(y), o.cols,
                 static_cast<float*>(vp_or_null(stats)), st(stream)),
        "norm");
  return {y, stats};
}

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w,
                        const OptTensor& b, const mxgg_norm_options& o, int64_t stream) {
    const variable_list r = norm_forward(x, w, b, o, true, stream);
    ctx->save_for_backward({x, w.value_or(Tensor()), r[1]});
    keep(ctx, "options", o);
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["need"] =
        (int64_t)(x.requires_grad() | grad_needed(w) << 1 | grad_needed(b) << 2);
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order("norm");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const auto o = kept<mxgg_norm_options>(ctx, "options");
    const int64_t need = ctx->saved_data["need"].toInt();
    Tensor dy = grads[0].to(x.scalar_type());
    if (row_stride(dy) < 0) dy = dy.contiguous();
    const auto param = [&](int bit, int32_t type) {
      return need & bit ? empty({o.cols}, x, type == MXGG_OUT_BF16 ? at::kBFloat16 : at::kFloat)
                        : Tensor();
    };
    Tensor dx = need & 1 ? empty(x.sizes(), x, x.scalar_type()) : Tensor();
    Tensor dw = param(2, o.weight_dtype), db = param(4, o.bias_dtype), ws;
    if (need & 6) ws = empty({lib.norm_grad_workspace_bytes(&o)}, x, at::kByte);
    check(lib.norm_grad(cp(dy), row_stride(dy), cp(x), row_stride(x), cp_or_null(w),
                        stats.const_data_ptr<float>(), &o, vp_or_null(dx), o.cols, vp_or_null(dw),
                        vp_or_null(db), vp_or_null(ws), ws.defined() ? ws.numel() : 0,
                        st(ctx->saved_data["stream"].toInt())),
          "norm_grad");
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

Result norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
            bool center, int64_t stream) {
  if (!plain(x) || !f32_or_bf16(x) || x.dim() < 1 || x.size(-1) > 32768 || row_stride(x) < 0 ||
      tangent(x) || tangent(weight) || tangent(bias))
    return none();
  const int64_t cols = x.size(-1);
  for (const OptTensor* p : {&weight, &bias})
    if (*p && (!plain(**p) || !f32_or_bf16(**p) || (*p)->dim() != 1 || (*p)->size(0) != cols ||
               !(*p)->is_contiguous() || (*p)->device() != x.device()))
      return none();
  const mxgg_norm_options o{x.numel() / cols,
                            cols,
                            type_of(x),
                            weight ? type_of(*weight) : MXGG_OUT_F32,
                            bias ? type_of(*bias) : MXGG_OUT_F32,
                            center,
                            (float)eps};
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || grad_needed(weight) || grad_needed(bias)))
    return Norm::apply(x, weight, bias, o, stream);
  return norm_forward(x, weight, bias, o, false, stream)[0];
}

// bf16 rows the loss kernels read in place.
bool loss_rows(const Tensor& t) {
  return plain(t) && t.scalar_type() == at::kBFloat16 && t.dim() >= 1 && row_stride(t) > 0 &&
         row_stride(t) % 8 == 0 && aligned(t.const_data_ptr(), 16);
}
// (loss, stats)
variable_list loss_forward(const Tensor& x, const Tensor& w, const Tensor& target,
                           const mxgg_loss_options& o, int64_t stream) {
  const bool each = o.reduction == MXGG_REDUCE_NONE;
  Tensor loss = each ? empty(target.sizes(), x, at::kFloat) : empty({}, x, at::kFloat);
  Tensor stats = empty({2 * o.tokens + 1}, x, at::kFloat);
  const int64_t bytes = lib.linear_cross_entropy_workspace_bytes(&o);
  Tensor ws = empty({std::max<int64_t>(bytes, 0)}, x, at::kByte);
  check(lib.linear_cross_entropy(cp(x), cp(w), cp(target), &o, loss.data_ptr<float>(),
                                 stats.data_ptr<float>(), vp(ws), bytes, st(stream)),
        "linear_cross_entropy");
  return {loss, stats};
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const Tensor& target, const mxgg_loss_options& o, int64_t stream) {
    const variable_list r = loss_forward(x, w, target, o, stream);
    ctx->save_for_backward({x, w, target, r[1]});
    keep(ctx, "options", o);
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (int)w.requires_grad() << 1);
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order("linear_cross_entropy");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &target = saved[2], &stats = saved[3];
    const auto o = kept<mxgg_loss_options>(ctx, "options");
    const int64_t need = ctx->saved_data["need"].toInt();
    const Tensor d = grads[0].to(at::kFloat).contiguous();
    Tensor dx, dw;
    if (need & 1) dx = empty(x.sizes(), x, x.scalar_type());
    if (need & 2) dw = empty(w.sizes(), w, w.scalar_type());
    const int64_t bytes =
        lib.linear_cross_entropy_grad_workspace_bytes(&o, (int)(need & 1), (int)(need & 2));
    Tensor ws = empty({std::max<int64_t>(bytes, 0)}, x, at::kByte);
    check(lib.linear_cross_entropy_grad(d.const_data_ptr<float>(), cp(x), cp(w), cp(target),
                                        stats.const_data_ptr<float>(), &o, vp_or_null(dx),
                                        vp_or_null(dw), vp(ws), bytes,
                                        st(ctx->saved_data["stream"].toInt())),
          "linear_cross_entropy_grad");
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

Result linear_cross_entropy(const Tensor& x, const Tensor& w, const Tensor& target,
                            int64_t ignore_index, int reduction, int64_t stream) {
  if (!loss_rows(x) || !loss_rows(w) || w.dim() != 2 || x.size(-1) != w.size(1) ||
      w.device() != x.device() || !plain(target) || !target.is_contiguous() ||
      (target.scalar_type() != at::kInt && target.scalar_type() != at::kLong) ||
      target.device() != x.device() || target.dim() != x.dim() - 1 ||
      target.sizes() != x.sizes().slice(0, x.dim() - 1) || tangent(x) || tangent(w))
    return none();
  const mxgg_loss_options o{target.numel(), w.size(0),    x.size(-1),
                            row_stride(x),  row_stride(w), ignore_index,
                            target.scalar_type() == at::kLong, reduction};
  if (lib.linear_cross_entropy_workspace_bytes(&o) < 0) return none();
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad()))
    return LinearCrossEntropy::apply(x, w, target, o, stream);
  return loss_forward(x, w, target, o, stream)[0];
}

// One AdamW step of lists of tensors; m_scales and v_scales are empty for 32-bit
// states, masters without master copies.
Result adamw(const std::vector<Tensor>& params, const std::vector<Tensor>& grads,
             const std::vector<Tensor>& m, const std::vector<Tensor>& v,
             const std::vector<Tensor>& m_scales, const std::vector<Tensor>& v_scales,
             const std::vector<Tensor>& masters, int64_t step, double lr, double beta1,
             double beta2, double eps, double weight_decay, int64_t stream) {
  const size_t n = params.size();
  const bool small = !m_scales.empty();
  if (n == 0 || grads.size() != n || m.size() != n || v.size() != n ||
      (small && (m_scales.size() != n || v_scales.size() != n)) ||
      (!masters.empty() && masters.size() != n))
    return none();
  const auto device = params[0].device();
  const auto ok = [&](const Tensor& t, int64_t numel) {
    return plain(t) && t.is_contiguous() && t.numel() == numel && t.device() == device;
  };
  const auto state_type = [&](const Tensor& t) {
    return small ? bytes(t) : t.scalar_type() == at::kFloat;
  };
  std::vector<mxgg_adamw_tensor> table(n);
  for (size_t i = 0; i < n; ++i) {
    const int64_t size = params[i].numel(), blocks = (size + 31) / 32;
    if (!ok(params[i], size) || !f32_or_bf16(params[i]) || !ok(grads[i], size) ||
        !f32_or_bf16(grads[i]) || !ok(m[i], size) || !state_type(m[i]) || !ok(v[i], size) ||
        !state_type(v[i]))
      return none();
    if (small && (!ok(m_scales[i], blocks) || m_scales[i].scalar_type() != at::kByte ||
                  !ok(v_scales[i], blocks) || v_scales[i].scalar_type() != at::kByte))
      return none();
    if (!masters.empty() && (!ok(masters[i], size) || masters[i].scalar_type() != at::kFloat))
      return none();
    table[i] = {vp(params[i]),
                cp(grads[i]),
                vp(m[i]),
                vp(v[i]),
                small ? vp(m_scales[i]) : nullptr,
                small ? vp(v_scales[i]) : nullptr,
                masters.empty() ? nullptr : masters[i].data_ptr<float>(),
                size,
                type_of(params[i]),
                type_of(grads[i])};
  }
  const mxgg_adamw_options o{lr, beta1, beta2, eps, weight_decay, step, small ? 8 : 32};
  const int rc = lib.adamw_step(table.data(), (int64_t)n, &o, st(stream));
  if (rc == MXGG_OK)  // modified in place, as far as torch and weight caches are concerned
    for (const auto* list : {&params, &m, &v, &m_scales, &v_scales, &masters})
      for (const Tensor& t : *list) t.unsafeGetTensorImpl()->bump_version();
  return rc;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("dim0", torch::wrap_pybind_function_no_gil(&dim0));
  m.def("dim1", torch::wrap_pybind_function_no_gil(&dim1));
  m.def("dual", torch::wrap_pybind_function_no_gil(&dual));
  m.def("mm", torch::wrap_pybind_function_no_gil(&mm));
  m.def("mm_swiglu", torch::wrap_pybind_function_no_gil(&mm_swiglu));
  m.def("wgrad", torch::wrap_pybind_function_no_gil(&wgrad));
  m.def("swiglu_bwd", torch::wrap_pybind_function_no_gil(&swiglu_bwd));
  m.def("zero_rows", torch::wrap_pybind_function_no_gil(&zero_rows));
  m.def("gather_dual", torch::wrap_pybind_function_no_gil(&gather_dual));
  m.def("gather_dim0", torch::wrap_pybind_function_no_gil(&gather_dim0));
  m.def("combine", torch::wrap_pybind_function_no_gil(&combine));
  m.def("route_topk", torch::wrap_pybind_function_no_gil(&route_topk));
  m.def("norm", torch::wrap_pybind_function_no_gil(&norm));
  m.def("linear_cross_entropy", torch::wrap_pybind_function_no_gil(&linear_cross_entropy));
  m.def("adamw", torch::wrap_pybind_function_no_gil(&adamw));
}
