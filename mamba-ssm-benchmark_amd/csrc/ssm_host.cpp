// Python binding of the launches (module ssm_scan._ssmhost): operand checks, output and workspace
// allocation and the argument structs of the C ABI in one call per launch.  The same work done from
// Python -- a ctypes struct of up to 25 views, 5-10 torch.empty calls, device and stream lookups --
// took 15-45 us per launch, more than the kernels of a short scan, a conv or a norm: rms_norm
// forward + backward (8192 x 256) 120 us against 18 us of kernels.
//
// Nothing here is numerical and nothing is kept between calls but a DecodePlan's weight tensors.
// Errors of the C ABI become the exception classes of ssm_scan._abi.check.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <atomic>
#include <optional>
#include <sstream>
#include <vector>

#include "../../include/ssm_scan.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// ------------------------------------------------------------------ helpers
ssm_tensor view(const Tensor &t) {
  ssm_tensor v{};
  if (!t.defined()) return v;
  TORCH_CHECK_VALUE(t.dim() <= 3, "expected a tensor of at most 3 dims, got ", t.dim());
  v.data = t.data_ptr();
  for (int64_t i = 0; i < t.dim(); ++i) v.stride[i] = t.stride(i);
  return v;
}
Tensor get(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
py::object out(const Tensor &t) { return t.defined() ? py::cast(t) : py::none(); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SSM_F32;
    case at::kBFloat16: return SSM_BF16;
    case at::kHalf: return SSM_F16;
    case at::kDouble: return SSM_F64;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t);
  }
}
bool io_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf || t == at::kDouble;
}

void check(int rc, const char *what) {
  if (rc == SSM_OK) return;
  TORCH_CHECK_VALUE(rc != SSM_EINVAL && rc != SSM_ESPACE, what, ": ", ssm_last_error());
  TORCH_CHECK(false, what, ": ", ssm_last_error());
}
// A *_bytes query: the check behind it names what is wrong.
#define SSM_BYTES(var, query, checkfn, args, what) \
  const int64_t var = query(&args);                \
  if (var < 0) {                                   \
    check(checkfn(&args), what);                   \
    check(SSM_EINVAL, what);                       \
  }

void require_gpu(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    TORCH_CHECK(!t->defined() || t->is_cuda(), "ssm_scan runs on ROCm GPU tensors only; got a tensor on ",
                t->device().str(), " (there is no CPU path)");
}

std::string shape_str(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}
void want(const char *name, const Tensor &t, at::IntArrayRef shape) {
  if (t.defined())
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape_str(shape), ", got ", shape_str(t.sizes()));
}

Tensor cast(const Tensor &t, at::ScalarType dt) { return !t.defined() || t.scalar_type() == dt ? t : t.to(dt); }
// Output buffer with t's layout when t is dense (e.g. channel-major views), else contiguous.
Tensor like(const Tensor &t, at::ScalarType dt) {
  const auto o = t.options().dtype(dt);
  return t.is_non_overlapping_and_dense() ? at::empty_like(t, o, at::MemoryFormat::Preserve) : at::empty(t.sizes(), o);
}
Tensor empty(at::IntArrayRef s, const Tensor &ref, at::ScalarType dt) { return at::empty(s, ref.options().dtype(dt)); }
Tensor bytes(int64_t n, const Tensor &ref) { return at::empty({std::max<int64_t>(n, 1)}, ref.options().dtype(at::kByte)); }

// profiling.KernelTimers in effect.
std::atomic<int> timers{0};

// The engine launches on the current device and on torch's current stream there.
struct Launch {
  c10::DeviceGuard guard;
  void *stream;
  explicit Launch(const Tensor &t)
      : guard(t.device()), stream((void *)c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
  // One launch, without the GIL: it blocks while the device's queue is full, and other Python threads
  // run on.  `timer` (a profiling.KernelTimer, or None) records its events right around it: the operand
  // checks, casts and allocations of the call are outside.
  template <typename Args>
  void run(const char *what, int (*fn)(const Args *, void *), const Args &args, const py::object &timer = py::none()) const {
    const py::object end = timer.is_none() ? timer : timer.attr("begin")(what);
    int rc;
    {
      py::gil_scoped_release release;
      rc = fn(&args, stream);
    }
    if (!end.is_none()) end.attr("record")();
    check(rc, what);
  }
  // The same from anywhere: a backward node runs on autograd's thread without the GIL, and waiting for it
  // there would cost a small backward a fifth of its time.  Only a timer needs it.
  template <typename Args>
  void run_anywhere(const char *what, int (*fn)(const Args *, void *), const Args &args) const {
    if (timers.load(std::memory_order_relaxed)) {
      const py::gil_scoped_acquire gil;
      return run(what, fn, args, py::module_::import("ssm_scan.profiling").attr("active")());
    }
    std::optional<py::gil_scoped_release> release;
    if (PyGILState_Check()) release.emplace();
    const int rc = fn(&args, stream);
    release.reset();
    check(rc, what);
  }
};

// ------------------------------------------------------------------ fused scan
void scan_checks(const Tensor &x, const OptTensor &delta_, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
                 const OptTensor &D_, const OptTensor &z_, const OptTensor &bias_, const OptTensor &h0_,
                 const OptTensor &proj_) {
  const Tensor delta = get(delta_), D = get(D_), z = get(z_), bias = get(bias_), h0 = get(h0_), proj = get(proj_);
  require_gpu({&x, &delta, &A, &Bm, &Cm, &D, &z, &bias, &h0, &proj});
  TORCH_CHECK_VALUE(x.dim() == 3, "x must be (B, L, D), got ", shape_str(x.sizes()));
  const int64_t B = x.size(0), L = x.size(1), Dm = x.size(2);
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == Dm, "A must be (D, N) = (", Dm, ", N), got ", shape_str(A.sizes()));
  const int64_t N = A.size(1);
  int64_t dd = Dm;
  if (proj.defined()) {
    TORCH_CHECK_VALUE(proj.dim() == 2 && proj.size(0) == Dm, "delta_proj must be (D, R) = (", Dm, ", R), got ",
                      shape_str(proj.sizes()));
    dd = proj.size(1);
  }
  want("delta", delta, {B, L, dd});
  want("Bm", Bm, {B, L, N});
  want("Cm", Cm, {B, L, N});
  want("D", D, {Dm});
  want("z", z, {B, L, Dm});
  want("delta_bias", bias, {Dm});
  want("h0", h0, {B, Dm, N});
}

template <typename Args>
void fill_scan(Args &a, const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
               const Tensor &D, const Tensor &z, const Tensor &bias, const Tensor &h0, const Tensor &proj, int method,
               bool softplus, bool a_log, int segments) {
  memset(&a, 0, sizeof(a));
  a.batch = x.size(0); a.seqlen = x.size(1); a.dim = x.size(2); a.dstate = A.size(1);
  a.method = method;
  a.dtype = dtype_code(x.scalar_type());
  a.x = view(x); a.delta = view(delta); a.A = view(A); a.Bm = view(Bm); a.Cm = view(Cm);
  a.Dskip = view(D); a.z = view(z); a.delta_bias = view(bias); a.h0 = view(h0);
  a.delta_softplus = softplus;
  a.segments = segments;
  if (proj.defined()) {
    a.delta_proj = view(proj);
    a.delta_rank = proj.size(1);
  }
  a.A_is_log = a_log;
}

// (out in the io dtype, last, the tensors scan_backward needs)
py::tuple scan_forward(const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
                       const OptTensor &D_, const OptTensor &z_, const OptTensor &bias_, const OptTensor &h0_, int method,
                       bool softplus, int segments, const OptTensor &proj_, bool a_log, bool need_saved, const py::object &timer) {
  at::ScalarType ct = c10::promoteTypes(x.scalar_type(), at::kFloat), io = at::kFloat;
  const Tensor z = get(z_);
  if (ct == at::kDouble) {
    io = ct;
  } else {
    ct = at::kFloat;
    bool same = io_type(x.scalar_type());
    for (const Tensor *t : {&delta, &Bm, &Cm, &z}) same = same && (!t->defined() || t->scalar_type() == x.scalar_type());
    if (same) io = x.scalar_type();
  }
  const Tensor xs = cast(x, io), ds = cast(delta, io), Bs = cast(Bm, io), Cs = cast(Cm, io), zs = cast(z, io);
  const Tensor As = cast(A, ct), Dv = cast(get(D_), ct), bv = cast(get(bias_), ct), h0 = cast(get(h0_), ct),
               W = cast(get(proj_), ct);
  const Tensor o = like(xs, io), last = empty({x.size(0), x.size(2), A.size(1)}, x, ct);
  ssm_fwd_args a;
  fill_scan(a, xs, ds, As, Bs, Cs, Dv, zs, bv, h0, W, method, softplus, a_log, segments);
  a.out = view(o);
  a.last = view(last);
  SSM_BYTES(wbytes, ssm_fwd_workspace_bytes, ssm_fwd_check, a, "ssm_fwd");
  Tensor ws, saved;
  if (wbytes) {
    ws = bytes(wbytes, x);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = wbytes;
  }
  if (need_saved) {
    SSM_BYTES(sbytes, ssm_fwd_saved_bytes, ssm_fwd_check, a, "ssm_fwd_saved_bytes");
    saved = bytes(sbytes, x);
    a.saved = saved.data_ptr();
  }
  const Launch l(x);
  l.run("ssm_fwd", ssm_fwd, a, timer);
  return py::make_tuple(o, last, py::make_tuple(xs, ds, As, Bs, Cs, out(Dv), out(zs), out(bv), out(h0), out(W), out(saved)));
}

py::tuple scan_backward(const Tensor &xs, const Tensor &ds, const Tensor &As, const Tensor &Bs, const Tensor &Cs,
                        const OptTensor &Dv_, const OptTensor &zs_, const OptTensor &bv_, const OptTensor &h0_,
                        const OptTensor &W_, const Tensor &saved, int method, bool softplus, bool a_log, int segments,
                        const OptTensor &dout_, const OptTensor &dlast_, const OptTensor &dz_, const OptTensor &dB_,
                        const OptTensor &dC_, const py::object &timer) {
  const Tensor Dv = get(Dv_), zs = get(zs_), bv = get(bv_), h0 = get(h0_), W = get(W_);
  const at::ScalarType io = xs.scalar_type(), ct = As.scalar_type();
  const Tensor dout = dout_ ? cast(*dout_, io) : at::zeros(xs.sizes(), xs.options());
  const Tensor dlast = cast(get(dlast_), ct);
  const int64_t B = xs.size(0), Dm = xs.size(2), N = As.size(1);
  const Tensor dx = like(xs, io), dd = like(W.defined() ? xs : ds, io), dA = empty({Dm, N}, xs, ct);
  const Tensor dB = dB_ ? *dB_ : like(Bs, io), dC = dC_ ? *dC_ : like(Cs, io);
  const Tensor dz = dz_ ? *dz_ : zs.defined() ? like(zs, io) : Tensor();
  const Tensor dD = Dv.defined() ? empty({Dm}, xs, ct) : Tensor(), db = bv.defined() ? empty({Dm}, xs, ct) : Tensor();
  const Tensor dh0 = h0.defined() ? empty({B, Dm, N}, xs, ct) : Tensor();
  ssm_bwd_args a;
  fill_scan(a, xs, ds, As, Bs, Cs, Dv, zs, bv, h0, W, method, softplus, a_log, segments);
  a.saved = saved.data_ptr();
  a.dout = view(dout); a.dlast = view(dlast);
  a.dx = view(dx); a.ddelta = view(dd); a.dA = view(dA);
  a.dBm = view(dB); a.dCm = view(dC); a.dD = view(dD);
  a.dz = view(dz); a.ddelta_bias = view(db); a.dh0 = view(dh0);
  SSM_BYTES(n, ssm_bwd_workspace_bytes, ssm_bwd_check, a, "ssm_bwd");
  const Tensor ws = bytes(n, xs);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  const Launch l(xs);
  l.run("ssm_bwd", ssm_bwd, a, timer);
  return py::make_tuple(dx, dd, dA, dB, dC, out(dD), out(dz), out(db), out(dh0));
}

// ------------------------------------------------------------------ conv
ssm_conv_args conv_args(const Tensor &x, const Tensor &w, const Tensor &bias, bool act) {
  ssm_conv_args a;
  memset(&a, 0, sizeof(a));
  a.batch = x.size(0); a.seqlen = x.size(1); a.dim = x.size(2); a.width = w.size(1);
  a.dtype = dtype_code(x.scalar_type());
  a.silu = act;
  a.x = view(x); a.weight = view(w); a.bias = view(bias);
  return a;
}

Tensor conv_forward(const Tensor &x, const Tensor &w, const OptTensor &bias, bool act, const OptTensor &state) {
  const Tensor o = at::empty(x.sizes(), x.options());
  ssm_conv_args a = conv_args(x, w, get(bias), act);
  a.out = view(o);
  if (state) a.state_in = a.state_out = view(*state);
  const Launch l(x);
  l.run("ssm_conv_fwd", ssm_conv_fwd, a);
  return o;
}

py::tuple conv_backward(const Tensor &x, const Tensor &w, const OptTensor &bias_, const Tensor &dout_, bool act,
                        const OptTensor &dx_) {
  const Tensor bias = get(bias_), dout = cast(dout_, x.scalar_type());
  const Tensor dx = dx_ ? *dx_ : at::empty(x.sizes(), x.options()), dw = at::empty_like(w);
  const Tensor db = bias.defined() ? at::empty_like(bias) : Tensor();
  ssm_conv_args a = conv_args(x, w, bias, act);
  a.dout = view(dout); a.dx = view(dx); a.dweight = view(dw); a.dbias = view(db);
  SSM_BYTES(n, ssm_conv_workspace_bytes, ssm_conv_check, a, "ssm_conv_bwd");
  const Tensor ws = bytes(n, x);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  const Launch l(x);
  l.run("ssm_conv_bwd", ssm_conv_bwd, a);
  return py::make_tuple(dx, dw, out(db));
}

// ------------------------------------------------------------------ RMSNorm
ssm_norm_args norm_args(const Tensor &x2, const Tensor &w, double eps) {
  ssm_norm_args a;
  memset(&a, 0, sizeof(a));
  a.rows = x2.size(0);
  a.dim = x2.size(1);
  a.dtype = dtype_code(x2.scalar_type());
  a.eps = eps;
  a.x = view(x2);
  a.weight = view(w);
  return a;
}
Tensor rows(const Tensor &t, int64_t C) {
  const Tensor r = t.reshape({-1, C});
  return r.stride(1) == 1 ? r : r.contiguous();
}

// (out, x as rows, weight, rstd)
py::tuple norm_forward(const Tensor &x, const Tensor &weight, double eps) {
  const Tensor x2 = rows(x, x.size(-1)), w = weight.contiguous();
  const Tensor o = at::empty(x2.sizes(), x.options()), rstd = at::empty({x2.size(0)}, x.options());
  ssm_norm_args a = norm_args(x2, w, eps);
  a.out = view(o);
  a.rstd = rstd.data_ptr();
  const Launch l(x);
  l.run("ssm_norm_fwd", ssm_norm_fwd, a);
  return py::make_tuple(o.view(x.sizes()), x2, w, rstd);
}

py::tuple norm_backward(const Tensor &x2, const Tensor &w, const Tensor &rstd, const Tensor &dout, double eps) {
  const Tensor dy = rows(cast(dout, x2.scalar_type()), x2.size(1));
  const Tensor dx = at::empty(x2.sizes(), x2.options()), dw = at::empty(w.sizes(), w.options());
  ssm_norm_args a = norm_args(x2, w, eps);
  a.rstd = rstd.data_ptr();
  a.dout = view(dy);
  a.dx = view(dx);
  a.dweight = dw.data_ptr();
  SSM_BYTES(n, ssm_norm_workspace_bytes, ssm_norm_check, a, "ssm_norm_bwd");
  const Tensor ws = bytes(n, x2);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  const Launch l(x2);
  l.run("ssm_norm_bwd", ssm_norm_bwd, a);
  return py::make_tuple(dx.view(dout.sizes()), dw);
}

// ------------------------------------------------------------------ linear scans
template <typename Args>
void fill_lscan(Args &args, const Tensor &a, int algo, int64_t chunk, bool reverse) {
  memset(&args, 0, sizeof(args));
  args.batch = a.size(0); args.seqlen = a.size(1); args.width = a.size(2);
  args.algo = algo;
  args.dtype = dtype_code(a.scalar_type());
  args.reverse = reverse;
  args.chunk = chunk;
}

Tensor lscan_forward(const Tensor &a, const Tensor &b, const OptTensor &h0, int algo, int64_t chunk, bool reverse,
                     const py::object &timer) {
  const Tensor h = at::empty(a.sizes(), a.options());
  ssm_lscan_args args;
  fill_lscan(args, a, algo, chunk, reverse);
  args.a = view(a); args.b = view(b); args.h0 = view(get(h0)); args.h = view(h);
  SSM_BYTES(n, ssm_lscan_workspace_bytes, ssm_lscan_check, args, "ssm_lscan");
  Tensor ws;
  if (n) {
    ws = bytes(n, a);
    args.workspace = ws.data_ptr();
    args.workspace_bytes = n;
  }
  const Launch l(a);
  l.run("ssm_lscan", ssm_lscan, args, timer);
  return h;
}

py::tuple lscan_backward(const Tensor &a, const OptTensor &h0_, const Tensor &h, const Tensor &dh, int algo, int64_t chunk,
                         bool reverse, bool need_dh0, const py::object &timer) {
  const Tensor h0 = get(h0_);
  const Tensor da = at::empty_like(h), db = at::empty_like(h);
  const Tensor dh0 = h0.defined() && need_dh0 ? at::empty_like(h0) : Tensor();
  ssm_lscan_bwd_args args;
  fill_lscan(args, a, algo, chunk, reverse);
  args.a = view(a); args.h0 = view(h0); args.h = view(h); args.dh = view(dh);
  args.da = view(da); args.db = view(db); args.dh0 = view(dh0);
  SSM_BYTES(n, ssm_lscan_bwd_workspace_bytes, ssm_lscan_bwd_check, args, "ssm_lscan_bwd");
  Tensor ws;
  if (n) {
    ws = bytes(n, a);
    args.workspace = ws.data_ptr();
    args.workspace_bytes = n;
  }
  const Launch l(a);
  l.run("ssm_lscan_bwd", ssm_lscan_bwd, args, timer);
  return py::make_tuple(da, db, out(dh0));
}

// ------------------------------------------------------------------ composed scan
constexpr int64_t kCscanWorkspace = 1LL << 28;  // bytes of dB / dC partials per backward launch
constexpr int64_t kCscanChannels = 1LL << 21;   // channels per launch

// t, or a contiguous copy where 64 steps of a batch row span 2 GiB (the kernels' offsets).
Tensor steps_fit(const Tensor &t) {
  const int64_t span = (t.stride(2) * (t.size(2) - 1) + 63 * t.stride(1) + 1) * t.element_size();
  return span < (1LL << 31) ? t : t.contiguous();
}
Tensor chans(const Tensor &t, int64_t dim, int64_t i, int64_t n) {
  return !t.defined() || (i == 0 && n == t.size(dim)) ? t : t.narrow(dim, i, n);
}

ssm_cscan_args cscan_args(const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
                          const Tensor &h0, const Tensor &saved, int64_t i, int64_t n, int algo, int method) {
  ssm_cscan_args a;
  memset(&a, 0, sizeof(a));
  a.batch = x.size(0); a.seqlen = x.size(1); a.dim = n; a.dstate = A.size(1);
  a.algo = algo;
  a.method = method;
  a.dtype = dtype_code(x.scalar_type());
  a.x = view(x); a.delta = view(delta); a.A = view(chans(A, 0, i, n)); a.Bm = view(Bm); a.Cm = view(Cm);
  a.h0 = view(chans(h0, 1, i, n));
  if (saved.defined()) {  // (B, tiles, D, N), states consecutive
    a.saved.data = (char *)saved.data_ptr() + i * saved.stride(2) * saved.element_size();
    for (int k = 0; k < 3; ++k) a.saved.stride[k] = saved.stride(k);
  }
  return a;
}

// (y, last, Bm, Cm, saved)
py::tuple cscan_forward(const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &Bm_, const Tensor &Cm_,
                        const OptTensor &h0_, int algo, int method, bool need_saved, const py::object &timer) {
  const Tensor Bm = steps_fit(Bm_), Cm = steps_fit(Cm_), h0 = get(h0_);
  const int64_t B = x.size(0), L = x.size(1), D = x.size(2), N = A.size(1);
  const Tensor y = at::empty_like(x), last = at::empty({B, D, N}, x.options());
  Tensor saved;
  if (need_saved) {
    const int64_t tile = ssm_cscan_tile(algo, dtype_code(x.scalar_type()));
    saved = at::empty({B, (L + tile - 1) / tile, D, N}, x.options());
  }
  const Launch l(x);
  for (int64_t i = 0; i < D || i == 0; i += kCscanChannels) {
    const int64_t n = std::min(D - i, kCscanChannels);
    const Tensor xb = steps_fit(chans(x, 2, i, n)), db = steps_fit(chans(delta, 2, i, n));
    ssm_cscan_args a = cscan_args(xb, db, A, Bm, Cm, h0, saved, i, n, algo, method);
    a.y = view(chans(y, 2, i, n));
    a.last = view(chans(last, 1, i, n));
    SSM_BYTES(nb, ssm_cscan_fwd_workspace_bytes, ssm_cscan_check, a, "ssm_cscan_fwd");
    Tensor ws;
    if (nb) {
      ws = bytes(nb, x);
      a.workspace = ws.data_ptr();
      a.workspace_bytes = nb;
    }
    l.run("ssm_cscan_fwd", ssm_cscan_fwd, a, timer);
  }
  return py::make_tuple(y, last, Bm, Cm, out(saved));
}

// Channel tiles of d_block, else all channels at once up to kCscanChannels and as many as keep the
// partials (2 x L x NP per 64 / NP channels and batch row) within kCscanWorkspace.
py::tuple cscan_backward(const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
                         const OptTensor &h0_, const Tensor &saved, int algo, int method, int64_t d_block,
                         const OptTensor &dy_, const OptTensor &dlast_, const py::object &timer) {
  const Tensor h0 = get(h0_), dlast = get(dlast_);
  const Tensor dy = dy_ ? *dy_ : at::zeros_like(x);
  const int64_t B = x.size(0), L = x.size(1), D = x.size(2), N = A.size(1);
  int64_t step = kCscanChannels;
  if (d_block > 0) {
    step = std::min(step, d_block);
  } else {
    const int64_t NP = N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64;
    step = std::min(step, std::max<int64_t>(1, kCscanWorkspace / (B * L * 2 * NP * x.element_size())) * (64 / NP));
  }
  const Tensor dx = at::empty_like(x), dd = at::empty_like(delta), dA = at::empty_like(A);
  const Tensor dh0 = h0.defined() ? at::empty_like(h0) : Tensor();
  Tensor dB, dC;
  const Launch l(x);
  for (int64_t i = 0; i < D; i += step) {
    const int64_t n = std::min(D - i, step);
    const Tensor gB = at::empty_like(Bm), gC = at::empty_like(Cm);
    const Tensor xb = steps_fit(chans(x, 2, i, n)), db = steps_fit(chans(delta, 2, i, n)), yb = steps_fit(chans(dy, 2, i, n));
    ssm_cscan_args a = cscan_args(xb, db, A, Bm, Cm, h0, saved, i, n, algo, method);
    a.dy = view(yb); a.dlast = view(chans(dlast, 1, i, n));
    a.dx = view(chans(dx, 2, i, n)); a.ddelta = view(chans(dd, 2, i, n)); a.dA = view(chans(dA, 0, i, n));
    a.dBm = view(gB); a.dCm = view(gC); a.dh0 = view(chans(dh0, 1, i, n));
    SSM_BYTES(nb, ssm_cscan_workspace_bytes, ssm_cscan_check, a, "ssm_cscan_bwd");
    const Tensor ws = bytes(nb, x);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = nb;
    l.run("ssm_cscan_bwd", ssm_cscan_bwd, a, timer);
    if (!dB.defined()) {
      dB = gB;
      dC = gC;
    } else {
      dB.add_(gB);
      dC.add_(gC);
    }
  }
  return py::make_tuple(dx, dd, dA, dB, dC, out(dh0));
}

// ------------------------------------------------------------------ gated delta rule
// t, or a contiguous copy where its last dimension is strided (the kernels read rows).
Tensor unit_last(const Tensor &t) {
  return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
ssm_tensor lead_view(const Tensor &t, int64_t n) {  // the first n strides; the last dimension is unit stride
  ssm_tensor v{};
  v.data = t.data_ptr();
  for (int64_t i = 0; i < n; ++i) v.stride[i] = t.stride(i);
  return v;
}
bool needs_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// A dual tensor need not require a gradient: without this its tangent would be left out where no node is made.
void no_tangents(std::initializer_list<const Tensor *> ts, const char *what) {
  for (const Tensor *t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}
// The gradients of a backward that has itself no derivative: under create_graph they carry a node over the inputs and
// the outputs' gradients that refuses, where without one they would pass for constants.
struct Twice : torch::autograd::Node {
  const char *what;
  Twice(const char *w, torch::autograd::edge_list next) : Node(std::move(next)), what(w) {}
  variable_list apply(variable_list &&) override {
    TORCH_CHECK(false, what, " cannot be differentiated twice");
  }
};
void not_twice(variable_list &d, const variable_list &douts, const char *what) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::edge_list next = torch::autograd::get_current_node()->next_edges();
  for (const torch::autograd::Edge &e : torch::autograd::collect_next_edges(douts)) next.push_back(e);
  const auto node = std::make_shared<Twice>(what, std::move(next));
  for (Tensor &t : d)
    if (t.defined()) torch::autograd::set_history(t, node);
}
void one_device(const Tensor &x, std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == x.device(), "tensors on ", x.device().str(), " and ", t->device().str());
}
bool delta_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

// Shapes and types of one call; `lead` = (B, L) of the chunked form, (B,) of the step.
void delta_checks(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta, const Tensor &h,
                  int64_t lead) {
  require_gpu({&q, &k, &v, &g, &beta, &h});
  no_tangents({&q, &k, &v, &g, &beta, &h}, "the gated delta rule");
  one_device(q, {&k, &v, &g, &beta, &h});
  const char *const form = lead == 2 ? "(B, L, H, D)" : "(B, H, D)";
  for (const Tensor *t : {&q, &k, &v})
    TORCH_CHECK_VALUE(t->dim() == lead + 2, "q, k and v must be ", form, ", got ", shape_str(t->sizes()));
  const auto dims = v.sizes().slice(0, lead);
  std::vector<int64_t> wq(dims.begin(), dims.end()), wg = wq, wh{v.size(0), v.size(lead), q.size(-1), v.size(-1)};
  wq.push_back(q.size(lead));
  wq.push_back(q.size(-1));
  wg.push_back(v.size(lead));
  want("q", q, wq);
  want("k", k, wq);
  want("g", g, wg);
  want("beta", beta, wg);
  want(lead == 2 ? "h0" : "h", h, wh);
  TORCH_CHECK_VALUE(q.size(lead) > 0 && v.size(lead) % q.size(lead) == 0, v.size(lead), " value heads are not a multiple of ",
                    q.size(lead), " key heads");
  for (const Tensor *t : {&q, &k, &v, &beta})
    TORCH_CHECK_TYPE(delta_type(t->scalar_type()), "the gated delta rule takes float32, bfloat16 or float16, got ",
                     t->scalar_type());
  TORCH_CHECK_TYPE(at::isFloatingType(g.scalar_type()), "g must be floating, got ", g.scalar_type());
}

template <typename Args>
void fill_delta(Args &a, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta, int64_t lead,
                double scale, bool qk_norm) {
  memset(&a, 0, sizeof(a));
  a.batch = v.size(0); a.key_heads = q.size(lead); a.heads = v.size(lead);
  a.key_dim = q.size(-1); a.value_dim = v.size(-1);
  a.dtype = dtype_code(v.scalar_type());
  a.beta_f32 = beta.scalar_type() == at::kFloat;
  a.qk_norm = qk_norm;
  a.scale = (float)scale;
  a.q = lead_view(q, lead + 1); a.k = lead_view(k, lead + 1); a.v = lead_view(v, lead + 1);
  a.g = view(g); a.beta = view(beta);
}
// The operands as the kernels read them: q, k and v of one type (float32 where they differ), rows of
// unit stride, g in float32, beta in float32 or that type.
struct DeltaOps {
  Tensor q, k, v, g, beta;
  DeltaOps(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g_, const Tensor &beta_) {
    const at::ScalarType io = q_.scalar_type() == v_.scalar_type() && k_.scalar_type() == v_.scalar_type() ? v_.scalar_type() : at::kFloat;
    q = unit_last(cast(q_, io)); k = unit_last(cast(k_, io)); v = unit_last(cast(v_, io));
    g = cast(g_, at::kFloat);
    beta = beta_.scalar_type() == io ? beta_ : cast(beta_, at::kFloat);
  }
};

// o, last (undefined unless wanted) and the tensors delta_backward needs
struct DeltaOut {
  Tensor o, last;
  variable_list saved;
};
DeltaOut delta_forward(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g_, const Tensor &beta_,
                       const OptTensor &h0_, double scale, bool qk_norm, bool want_last, bool need_saved) {
  delta_checks(q_, k_, v_, g_, beta_, get(h0_), 2);
  const DeltaOps t(q_, k_, v_, g_, beta_);
  Tensor h0 = cast(get(h0_), at::kFloat);
  if (h0.defined()) h0 = h0.contiguous();
  const Tensor o = at::empty(t.v.sizes(), t.v.options());
  Tensor last, saved;
  if (want_last) last = empty({t.v.size(0), t.v.size(2), t.q.size(3), t.v.size(3)}, t.v, at::kFloat);
  ssm_delta_args a;
  fill_delta(a, t.q, t.k, t.v, t.g, t.beta, 2, scale, qk_norm);
  a.seqlen = t.v.size(1);
  a.h0 = h0.defined() ? h0.data_ptr<float>() : nullptr;
  a.out = lead_view(o, 3);
  a.last = last.defined() ? last.data_ptr<float>() : nullptr;
  SSM_BYTES(n, ssm_delta_fwd_workspace_bytes, ssm_delta_check, a, "ssm_delta_fwd");
  const Tensor ws = bytes(n, o);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  if (need_saved) {
    saved = bytes(ssm_delta_saved_bytes(&a), o);
    a.saved = saved.data_ptr();
  }
  const Launch l(o);
  l.run_anywhere("ssm_delta_fwd", ssm_delta_fwd, a);
  return {cast(o, v_.scalar_type()), last, {t.q, t.k, t.v, t.g, t.beta, saved}};
}

// dq, dk, dv, dg, dbeta, dh0 (undefined unless needed)
variable_list delta_backward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta,
                             const Tensor &saved, const Tensor &dout_, const Tensor &dlast_, double scale, bool qk_norm,
                             bool need_dh0) {
  const Tensor dout = dout_.defined() ? unit_last(cast(dout_, v.scalar_type())) : at::zeros(v.sizes(), v.options());
  Tensor dlast = cast(dlast_, at::kFloat);
  if (dlast.defined()) dlast = dlast.contiguous();
  auto dense = [](const Tensor &t) { return at::empty(t.sizes(), t.options()); };
  const Tensor dq = dense(q), dk = dense(k), dv = dense(v), dg = dense(g), db = dense(beta);
  Tensor dh0;
  if (need_dh0) dh0 = empty({v.size(0), v.size(2), q.size(3), v.size(3)}, v, at::kFloat);
  ssm_delta_args a;
  fill_delta(a, q, k, v, g, beta, 2, scale, qk_norm);
  a.seqlen = v.size(1);
  a.saved = saved.data_ptr();
  a.dout = lead_view(dout, 3);
  a.dlast = dlast.defined() ? dlast.data_ptr<float>() : nullptr;
  a.dq = lead_view(dq, 3); a.dk = lead_view(dk, 3); a.dv = lead_view(dv, 3);
  a.dg = view(dg); a.dbeta = view(db);
  a.dh0 = dh0.defined() ? dh0.data_ptr<float>() : nullptr;
  SSM_BYTES(n, ssm_delta_bwd_workspace_bytes, ssm_delta_check, a, "ssm_delta_bwd");
  const Tensor ws = bytes(n, v);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = n;
  const Launch l(v);
  l.run_anywhere("ssm_delta_bwd", ssm_delta_bwd, a);
  return {dq, dk, dv, dg, db, dh0};
}

// The rule's node in autograd, which runs without the interpreter.
struct DeltaFn : torch::autograd::Function<DeltaFn> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g,
                               const Tensor &beta, const OptTensor &h0, double scale, bool qk_norm, bool want_last) {
    DeltaOut r = delta_forward(q, k, v, g, beta, h0, scale, qk_norm, want_last, true);
    ctx->save_for_backward(r.saved);
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["qk_norm"] = qk_norm;
    ctx->saved_data["h0"] = h0.has_value();
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)q.scalar_type(), (int64_t)k.scalar_type(), (int64_t)v.scalar_type(),
                                                    (int64_t)g.scalar_type(), (int64_t)beta.scalar_type(),
                                                    (int64_t)(h0 ? h0->scalar_type() : at::kFloat)};
    return want_last ? variable_list{r.o, r.last} : variable_list{r.o};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor dlast = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dlast.defined()) return variable_list(9);
    const variable_list t = ctx->get_saved_variables();
    variable_list d = delta_backward(t[0], t[1], t[2], t[3], t[4], t[5], grads[0], dlast, ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["qk_norm"].toBool(),
                                     ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(5));
    const auto types = ctx->saved_data["types"].toIntVector();
    for (size_t i = 0; i < d.size(); ++i) d[i] = cast(d[i], (at::ScalarType)types[i]);
    not_twice(d, grads, "the gated delta rule");
    d.resize(9);
    return d;
  }
};
// (o, last or None)
py::tuple delta(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta, const OptTensor &h0,
                double scale, bool qk_norm, bool want_last) {
  if (!needs_grad({&q, &k, &v, &g, &beta}) && !(h0 && needs_grad({&*h0}))) {
    const DeltaOut r = delta_forward(q, k, v, g, beta, h0, scale, qk_norm, want_last, false);
    return py::make_tuple(r.o, out(r.last));
  }
  const variable_list r = DeltaFn::apply(q, k, v, g, beta, h0, scale, qk_norm, want_last);
  return py::make_tuple(r[0], want_last ? py::cast(r[1]) : py::none());
}

Tensor delta_step(const Tensor &h, const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g_, const Tensor &beta_,
                  double scale, bool qk_norm) {
  delta_checks(q_, k_, v_, g_, beta_, h, 1);
  TORCH_CHECK_VALUE(h.scalar_type() == at::kFloat && h.is_contiguous(), "the state must be contiguous float32, got ",
                    h.scalar_type(), " with strides ", h.strides());
  TORCH_CHECK(!needs_grad({&h, &q_, &k_, &v_, &g_, &beta_}),
              "gated_delta_step is not differentiable, as it updates its state in place: call it under torch.no_grad()");
  if (h.size(0) == 0) return at::empty(v_.sizes(), v_.options());  // no stream
  const DeltaOps t(q_, k_, v_, g_, beta_);
  const Tensor o = at::empty(t.v.sizes(), t.v.options());
  ssm_delta_step_args a;
  fill_delta(a, t.q, t.k, t.v, t.g, t.beta, 1, scale, qk_norm);
  a.h = h.data_ptr<float>();
  a.out = lead_view(o, 2);
  const Launch l(o);
  l.run_anywhere("ssm_delta_step", ssm_delta_step, a);
  if (!h.is_inference()) h.unsafeGetTensorImpl()->bump_version();
  return o.scalar_type() == v_.scalar_type() ? o : o.to(v_.scalar_type());
}

// ------------------------------------------------------------------ grouped norm
ssm_gnorm_args gnorm_args(const Tensor &x2, const Tensor &w, const Tensor &b, const Tensor &gate2, int64_t groups, int act,
                          bool center, double eps) {
  ssm_gnorm_args a;
  memset(&a, 0, sizeof(a));
  a.rows = x2.size(0);
  a.groups = groups;
  a.group_size = x2.size(1) / groups;
  a.dtype = dtype_code(x2.scalar_type());
  a.activation = act;
  a.center = center;
  a.eps = eps;
  a.x = view(x2);
  a.gate = view(gate2);
  a.weight = w.defined() ? w.data_ptr<float>() : nullptr;
  a.bias = b.defined() ? b.data_ptr<float>() : nullptr;
  return a;
}
Tensor f32(const OptTensor &t) { return t ? cast(*t, at::kFloat).contiguous() : Tensor(); }

void gnorm_checks(const Tensor &x, const Tensor &w_, const Tensor &b_, const Tensor &g, int64_t groups) {
  require_gpu({&x, &g, &w_, &b_});
  one_device(x, {&g, &w_, &b_});
  no_tangents({&x, &g, &w_, &b_}, "group_norm");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0 && groups > 0 && x.size(-1) % groups == 0, "the last dimension of x, ",
                    shape_str(x.sizes()), ", is not ", groups, " whole groups");
  TORCH_CHECK_TYPE(delta_type(x.scalar_type()), "group_norm takes float32, bfloat16 or float16, got ", x.scalar_type());
  want("weight", w_, {x.size(-1)});
  want("bias", b_, {x.size(-1)});
  want("gate", g, x.sizes());
}
// y, x as rows, weight, bias, gate as rows
variable_list gnorm_forward(const Tensor &x, const OptTensor &weight, const OptTensor &bias, const OptTensor &gate,
                            int64_t groups, int64_t act, bool center, double eps) {
  const Tensor g = get(gate);
  const Tensor x2 = rows(x, x.size(-1)), w = f32(weight), b = f32(bias);
  const Tensor g2 = g.defined() ? rows(cast(g, x.scalar_type()), x.size(-1)) : g;
  const Tensor o = at::empty(x2.sizes(), x2.options());
  ssm_gnorm_args a = gnorm_args(x2, w, b, g2, groups, act, center, eps);
  a.out = view(o);
  const Launch l(x);
  l.run_anywhere("ssm_gnorm_fwd", ssm_gnorm_fwd, a);
  return {o.view(x.sizes()), x2, w, b, g2};
}

// dx, dweight, dbias, dgate, the last three undefined where their operand is
variable_list gnorm_backward(const Tensor &x2, const Tensor &w, const Tensor &b, const Tensor &g2, const Tensor &dout,
                             int64_t groups, int64_t act, bool center, double eps, bool need_dw, bool need_db) {
  const Tensor dy = rows(cast(dout, x2.scalar_type()), x2.size(1));
  const Tensor dx = at::empty(x2.sizes(), x2.options());
  const Tensor dgate = g2.defined() ? at::empty(x2.sizes(), x2.options()) : g2;
  const Tensor dw = need_dw ? empty({x2.size(1)}, x2, at::kFloat) : Tensor();
  const Tensor db = need_db ? empty({x2.size(1)}, x2, at::kFloat) : Tensor();
  ssm_gnorm_args a = gnorm_args(x2, w, b, g2, groups, act, center, eps);
  a.dout = view(dy);
  a.dx = view(dx);
  a.dgate = view(dgate);
  a.dweight = need_dw ? dw.data_ptr<float>() : nullptr;
  a.dbias = need_db ? db.data_ptr<float>() : nullptr;
  SSM_BYTES(n, ssm_gnorm_workspace_bytes, ssm_gnorm_check, a, "ssm_gnorm_bwd");
  Tensor ws;
  if (n) {
    ws = bytes(n, x2);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = n;
  }
  const Launch l(x2);
  l.run_anywhere("ssm_gnorm_bwd", ssm_gnorm_bwd, a);
  return {dx.view(dout.sizes()), dw, db, g2.defined() ? dgate.view(dout.sizes()) : g2};
}

struct GnormFn : torch::autograd::Function<GnormFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight, const OptTensor &bias,
                        const OptTensor &gate, int64_t groups, int64_t act, bool center, double eps) {
    const variable_list r = gnorm_forward(x, weight, bias, gate, groups, act, center, eps);
    ctx->save_for_backward({r[1], r[2], r[3], r[4]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->saved_data["center"] = center;
    ctx->saved_data["eps"] = eps;
    auto type = [&](const OptTensor &t) { return (int64_t)(t ? t->scalar_type() : at::kFloat); };
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), type(weight), type(bias), type(gate)};
    return r[0];
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list t = ctx->get_saved_variables();
    // edges are numbered over the tensors that were given
    const bool dw = t[1].defined() && ctx->needs_input_grad(1);
    const bool db = t[2].defined() && ctx->needs_input_grad(t[1].defined() ? 2 : 1);
    variable_list d = gnorm_backward(t[0], t[1], t[2], t[3], grads[0], ctx->saved_data["groups"].toInt(),
                                     ctx->saved_data["act"].toInt(), ctx->saved_data["center"].toBool(),
                                     ctx->saved_data["eps"].toDouble(), dw, db);
    const auto types = ctx->saved_data["types"].toIntVector();
    for (size_t i = 0; i < d.size(); ++i) d[i] = cast(d[i], (at::ScalarType)types[i]);
    not_twice(d, grads, "group_norm");
    d.resize(8);
    return d;
  }
};
Tensor gnorm(const Tensor &x, const OptTensor &weight, const OptTensor &bias, const OptTensor &gate, int64_t groups, int64_t act,
             bool center, double eps) {
  const Tensor w = get(weight), b = get(bias), g = get(gate);
  gnorm_checks(x, w, b, g, groups);
  if (x.numel() == 0) {  // no rows: an empty tensor in the graph of what was given
    Tensor y = x * 1;
    for (const Tensor *t : {&w, &b, &g})
      if (t->defined()) y = y * *t;
    return cast(y, x.scalar_type());
  }
  if (!needs_grad({&x, &w, &b, &g})) return gnorm_forward(x, weight, bias, gate, groups, act, center, eps)[0];
  return GnormFn::apply(x, weight, bias, gate, groups, act, center, eps);
}

// ------------------------------------------------------------------ decode
// The weights of a block stack's token step, laid out once; a step brings tokens and states.
struct DecodePlan {
  struct Block {
    Tensor w_in4, conv_w, conv_b, x_proj_wt, dt_proj_w, dt_bias, A_log, Dskip, w_out4;
    double eps;
  };
  std::vector<Block> blocks;
  Tensor head_w4;
  int64_t dm, dim, N, W, R, V;

  DecodePlan(const std::vector<std::pair<std::vector<Tensor>, double>> &layers, Tensor head, int64_t dm_, int64_t dim_,
             int64_t N_, int64_t W_, int64_t R_, int64_t V_)
      : head_w4(std::move(head)), dm(dm_), dim(dim_), N(N_), W(W_), R(R_), V(V_) {
    for (const auto &l : layers) {
      const auto &t = l.first;
      TORCH_CHECK_VALUE(t.size() == 9, "a decode block has 9 weights");
      blocks.push_back({t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], l.second});
    }
  }

  // Host-side checks before any launch: the kernels size every state buffer from the token count
  // and the model's dimensions.
  void check_states(const Tensor &tok, const std::vector<Tensor> &conv, const std::vector<Tensor> &ssm) const {
    const Tensor &w = blocks.at(0).w_in4;
    require_gpu({&w, &tok});
    for (size_t i = 0; i < conv.size(); ++i) require_gpu({&conv[i], &ssm[i]});
    const int64_t B = tok.numel();
    const auto dev = w.device();
    TORCH_CHECK_VALUE(tok.device() == dev, "tokens on ", tok.device().str(), ", the model on ", dev.str());
    TORCH_CHECK_VALUE(conv.size() == blocks.size(), conv.size(), " states for ", blocks.size(), " blocks");
    for (size_t i = 0; i < conv.size(); ++i) {
      const Tensor &c = conv[i], &s = ssm[i];
      const std::vector<int64_t> ws{B, dim, N}, wc{B, dim, W - 1};
      TORCH_CHECK_VALUE(s.sizes() == at::IntArrayRef(ws) && c.sizes() == at::IntArrayRef(wc), "block ", i, ": states ",
                        shape_str(s.sizes()), " / ", shape_str(c.sizes()), ", expected ", shape_str(ws), " / ",
                        shape_str(wc), " for ", B, " tokens");
      TORCH_CHECK_VALUE(s.device() == dev && c.device() == dev, "block ", i, ": states on ", s.device().str(), " / ",
                        c.device().str(), ", the model on ", dev.str());
      TORCH_CHECK_VALUE(c.is_contiguous() && s.is_contiguous() && s.scalar_type() == at::kFloat &&
                            (c.scalar_type() == at::kFloat || c.scalar_type() == at::kBFloat16),
                        "decode states must be contiguous: ssm float32, conv float32 or bf16");
    }
  }

  void fill(ssm_decode_stack_args &a, int64_t B) const {
    memset(&a, 0, sizeof(a));
    a.batch = B; a.dim = dim; a.dstate = N; a.width = W; a.dt_rank = R; a.d_model = dm;
    a.n_blocks = (int32_t)blocks.size();
    a.vocab = V;
  }
  int64_t workspace_bytes(int64_t B) const {
    ssm_decode_stack_args a;
    fill(a, B);
    return ssm_decode_stack_workspace_bytes(&a);
  }
  int64_t status_offset(int64_t B) const {
    ssm_decode_stack_args a;
    fill(a, B);
    return ssm_decode_stack_status_offset(&a);
  }

  // The whole token step in one call; returns the logits.  The discretization and the final norm's eps
  // are settings of the model, not weights: they come with each step.
  Tensor step(const Tensor &tok_, const std::vector<Tensor> &conv, const std::vector<Tensor> &ssm, const Tensor &embed,
              const Tensor &ws, int method, double head_eps) const {
    for (const Tensor &c : conv)
      TORCH_CHECK_VALUE(c.scalar_type() == conv[0].scalar_type(),
                        "the stack path needs one conv state dtype for every block");
    const Tensor tok = tok_.reshape({-1}).to(at::kLong).contiguous();  // a strided view of ids is copied
    const int64_t B = tok.numel();
    const auto f = head_w4.options();
    const Tensor u = at::empty({B, dm}, f), logits = at::empty({B, V}, f);
    std::vector<ssm_decode_block> k(blocks.size());
    auto p = [](const Tensor &t) { return (const float *)t.data_ptr(); };
    for (size_t i = 0; i < k.size(); ++i) {
      const Block &b = blocks[i];
      memset(&k[i], 0, sizeof(k[i]));
      k[i].w_in4 = p(b.w_in4); k[i].conv_w = p(b.conv_w); k[i].conv_b = p(b.conv_b); k[i].x_proj_wt = p(b.x_proj_wt);
      k[i].dt_proj_w = p(b.dt_proj_w); k[i].dt_bias = p(b.dt_bias); k[i].A_log = p(b.A_log); k[i].Dskip = p(b.Dskip);
      k[i].w_out4 = p(b.w_out4);
      k[i].conv_state = conv[i].data_ptr();
      k[i].ssm_state = (float *)ssm[i].data_ptr();
      k[i].eps = (float)b.eps;
    }
    ssm_decode_stack_args a;
    fill(a, B);
    a.method = method;
    a.head_eps = (float)head_eps;
    a.conv_state_dtype = dtype_code(conv[0].scalar_type());
    a.blocks = k.data();
    a.u = (float *)u.data_ptr();
    a.tokens = (const int64_t *)tok.data_ptr();
    a.embed = p(embed);
    a.head_w4 = p(head_w4);
    a.logits = (float *)logits.data_ptr();
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.numel();
    const Launch l(u);
    l.run("ssm_decode_stack", ssm_decode_stack, a);
    return logits;
  }
};

}  // namespace

PYBIND11_MODULE(_ssmhost, m) {
  m.def("scan_checks", torch::wrap_pybind_function(scan_checks));
  m.def("scan_forward", torch::wrap_pybind_function(scan_forward));
  m.def("scan_backward", torch::wrap_pybind_function(scan_backward));
  m.def("conv_forward", torch::wrap_pybind_function(conv_forward));
  m.def("conv_backward", torch::wrap_pybind_function(conv_backward));
  m.def("norm_forward", torch::wrap_pybind_function(norm_forward));
  m.def("norm_backward", torch::wrap_pybind_function(norm_backward));
  m.def("lscan_forward", torch::wrap_pybind_function(lscan_forward));
  m.def("lscan_backward", torch::wrap_pybind_function(lscan_backward));
  m.def("cscan_forward", torch::wrap_pybind_function(cscan_forward));
  m.def("cscan_backward", torch::wrap_pybind_function(cscan_backward));
  m.def("delta_checks", [](const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &beta,
                           const OptTensor &h) { delta_checks(q, k, v, g, beta, get(h), 2); });
  m.def("count_timers", [](int change) { timers += change; });
  m.def("delta", torch::wrap_pybind_function(delta));
  m.def("delta_step", torch::wrap_pybind_function(delta_step));
  m.def("gnorm", torch::wrap_pybind_function(gnorm));
  m.attr("ABI_VERSION") = SSM_ABI_VERSION;  // of the header the argument structs above were compiled from
  py::class_<DecodePlan>(m, "DecodePlan")
      .def(py::init<const std::vector<std::pair<std::vector<Tensor>, double>> &, Tensor, int64_t, int64_t, int64_t, int64_t,
                    int64_t, int64_t>())
      .def("check_states", torch::wrap_pybind_function(&DecodePlan::check_states))
      .def("workspace_bytes", &DecodePlan::workspace_bytes)
      .def("status_offset", &DecodePlan::status_offset)
      .def("step", torch::wrap_pybind_function(&DecodePlan::step));
}
