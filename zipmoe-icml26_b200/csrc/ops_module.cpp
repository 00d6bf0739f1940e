// Python module `zmoe._ops`: the torch-facing side of the sort, its gradients
// and the adapters, over the C ABI of libzmoe.so.  These calls run once per layer
// and token step, where the host's time counts: checking ten tensors, allocating
// outputs and filling an argument structure took 10 to 14 us in Python with
// ctypes and takes 2 to 4 here.  zmoe/ops.py documents each function.
//
// Bad arguments raise ValueError; a status other than ZMOE_OK raises
// zmoe._lib.ZmoeError with the library's message.  Work runs on the arguments'
// device and that device's current torch stream.
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>
#include <string>
#include <tuple>

#include "zmoe.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr auto kBF16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;
constexpr auto kI32 = at::kInt;

[[noreturn]] void value_error(const std::string& what) { throw py::value_error(what); }

std::string text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + ")";
}

// Device pointer of an argument after checking its type, shape and place.
template <class T>
T* arg(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  if (t.scalar_type() != type || t.sizes() != shape || t.device() != device || !t.is_contiguous())
    value_error(std::string(name) + ": expected a contiguous " + c10::toString(type) + " tensor of shape " + text(shape) +
                " on " + device.str() + ", got " + c10::toString(t.scalar_type()) + " " + text(t.sizes()) +
                (t.is_contiguous() ? "" : " (not contiguous)") + " on " + t.device().str());
  return static_cast<T*>(t.data_ptr());
}
template <class T>
T* arg(const OptTensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  return t ? arg<T>(*t, name, type, shape, device) : nullptr;
}

void dims(const Tensor& t, const char* name, int64_t n) {
  if (t.dim() != n) value_error(std::string(name) + ": expected " + std::to_string(n) + " dimensions, got " + std::to_string(t.dim()));
}

at::Device cuda(const Tensor& t, const char* name, int64_t n) {
  if (!t.is_cuda()) value_error(std::string(name) + ": expected a CUDA tensor");
  dims(t, name, n);
  return t.device();
}

int to_int(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) value_error(std::string(name) + ": size " + std::to_string(v) + " is too large");
  return static_cast<int>(v);
}

// An output, without at::empty's way through the dispatcher (0.3 us each).
Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
}

py::object* g_error = nullptr;                         // zmoe._lib.ZmoeError

// Calls an entry point with the GIL released.
template <class F>
void call(const char* what, at::Device device, F&& f) {
  c10::cuda::CUDAGuard guard(device);
  const auto stream = reinterpret_cast<zmoe_stream_t>(c10::cuda::getCurrentCUDAStream(device.index()).stream());
  zmoe_status st;
  {
    py::gil_scoped_release release;
    st = f(stream);
  }
  if (st != ZMOE_OK) {
    const std::string text = std::string(what) + ": status " + std::to_string(st) + ": " + zmoe_last_error();
    PyErr_SetString(g_error->ptr(), text.c_str());
    throw py::error_already_set();
  }
}

py::tuple permute(const Tensor& idx, const OptTensor& x, int64_t E, int64_t capacity, int64_t seq_len) {
  const at::Device dev = cuda(idx, "topk_idx", 2);
  const int64_t T = idx.size(0), k = idx.size(1);
  zmoe_permute_args a{};
  a.topk_idx = arg<int32_t>(idx, "topk_idx", kI32, {T, k}, dev);
  if (x) {
    // rows behind the last token may be there (a buffer for the largest batch) and are not read
    if (!x->is_cuda() || x->dim() != 2 || x->size(0) < T || x->scalar_type() != kBF16 || !x->is_contiguous() || x->device() != dev)
      value_error("x: expected a contiguous CUDA BF16 tensor with a row for each token");
    a.x = static_cast<const uint16_t*>(x->data_ptr());
    a.H = to_int(x->size(1), "H");
  }
  if (E < 1) value_error("E must be at least 1");
  a.T = to_int(T, "T");
  a.k = to_int(k, "k");
  a.E = to_int(E, "E");
  to_int(T * k, "T * k");
  a.capacity = to_int(capacity, "capacity");
  a.seq_len = to_int(seq_len, "seq_len");
  const int64_t rows = std::max<int64_t>(T * k, 1);
  Tensor counts = empty({E}, kI32, dev), offsets = empty({E + 1}, kI32, dev), row_of = empty({T, k}, kI32, dev),
         tor = empty({rows}, kI32, dev);
  py::object xp = py::none();
  if (x) {
    Tensor t = empty({rows, (int64_t)a.H}, kBF16, dev);
    a.xp = static_cast<uint16_t*>(t.data_ptr());
    xp = py::cast(t);
  }
  a.counts = static_cast<int32_t*>(counts.data_ptr());
  a.offsets = static_cast<int32_t*>(offsets.data_ptr());
  a.row_of = static_cast<int32_t*>(row_of.data_ptr());
  a.token_of_row = static_cast<int32_t*>(tor.data_ptr());
  call("zmoe_permute", dev, [&](zmoe_stream_t s) { return zmoe_permute(&a, s); });
  return py::make_tuple(counts, offsets, row_of, tor, xp);
}

Tensor permute_grad(const Tensor& dxp, const Tensor& row_of, const OptTensor& base, const OptTensor& dx_) {
  const at::Device dev = cuda(dxp, "dxp", 2);
  dims(row_of, "row_of", 2);
  const int64_t rows = dxp.size(0), H = dxp.size(1), T = row_of.size(0), k = row_of.size(1);
  zmoe_permute_grad_args a{};
  a.dxp = arg<uint16_t>(dxp, "dxp", kBF16, {rows, H}, dev);
  a.row_of = arg<int32_t>(row_of, "row_of", kI32, {T, k}, dev);
  a.base = arg<uint16_t>(base, "base", kBF16, {T, H}, dev);
  a.T = to_int(T, "T");
  a.H = to_int(H, "H");
  a.k = to_int(k, "k");
  a.rows = to_int(rows, "rows");
  Tensor dx = dx_ ? *dx_ : empty({T, H}, kBF16, dev);
  a.dx = arg<uint16_t>(dx, "dx", kBF16, {T, H}, dev);
  call("zmoe_permute_grad", dev, [&](zmoe_stream_t s) { return zmoe_permute_grad(&a, s); });
  return dx;
}

py::tuple combine_grad(const Tensor& dout, const Tensor& y, const Tensor& row_of, const Tensor& w, int64_t mode,
                       const OptTensor& y_shared, const OptTensor& shared_gate, const OptTensor& x, const OptTensor& dy_) {
  const at::Device dev = cuda(dout, "dout", 2);
  dims(y, "y", 2);
  dims(row_of, "row_of", 2);
  const int64_t T = dout.size(0), H = dout.size(1), rows = y.size(0), k = row_of.size(1);
  if (shared_gate && !y_shared) value_error("shared_gate without y_shared");
  if (mode == ZMOE_ROUTE_SWITCH && !x) value_error("x: Switch needs it");
  zmoe_combine_grad_args a{};
  a.dout = arg<uint16_t>(dout, "dout", kBF16, {T, H}, dev);
  a.y = arg<uint16_t>(y, "y", kBF16, {rows, H}, dev);
  a.y_shared = arg<uint16_t>(y_shared, "y_shared", kBF16, {T, H}, dev);
  a.shared_gate = arg<float>(shared_gate, "shared_gate", kF32, {T}, dev);
  a.row_of = arg<int32_t>(row_of, "row_of", kI32, {T, k}, dev);
  a.topk_w = arg<float>(w, "topk_w", kF32, {T, k}, dev);
  a.x = arg<uint16_t>(x, "x", kBF16, {T, H}, dev);
  a.T = to_int(T, "T");
  a.H = to_int(H, "H");
  a.k = to_int(k, "k");
  a.mode = to_int(mode, "mode");
  a.rows = to_int(rows, "rows");
  Tensor dy = dy_ ? *dy_ : empty({rows, H}, kBF16, dev), dw = empty({T, k}, kF32, dev);
  a.dy = arg<uint16_t>(dy, "dy", kBF16, {rows, H}, dev);
  a.dtopk_w = static_cast<float*>(dw.data_ptr());
  py::object dysh = py::none(), dg = py::none(), dx = py::none();
  if (y_shared) {
    Tensor t = empty({T, H}, kBF16, dev);
    a.dy_shared = static_cast<uint16_t*>(t.data_ptr());
    dysh = py::cast(t);
  }
  if (shared_gate) {
    Tensor t = empty({T}, kF32, dev);
    a.dshared_gate = static_cast<float*>(t.data_ptr());
    dg = py::cast(t);
  }
  if (mode == ZMOE_ROUTE_SWITCH) {
    Tensor t = empty({T, H}, kBF16, dev);
    a.dx = static_cast<uint16_t*>(t.data_ptr());
    dx = py::cast(t);
  }
  call("zmoe_combine_grad", dev, [&](zmoe_stream_t s) { return zmoe_combine_grad(&a, s); });
  return py::make_tuple(dy, dw, dysh, dg, dx);
}

py::tuple lora_plan(const Tensor& adapter, int64_t G) {
  const at::Device dev = cuda(adapter, "adapter", 1);
  const int64_t T = adapter.size(0);
  const int32_t* ids = arg<int32_t>(adapter, "adapter", kI32, {T}, dev);
  const int g = to_int(G, "G"), t = to_int(T, "T");
  Tensor offsets = empty({std::max<int64_t>(G, 0) + 1}, kI32, dev), tor = empty({T}, kI32, dev);
  auto* po = static_cast<int32_t*>(offsets.data_ptr());
  auto* pt = static_cast<int32_t*>(tor.data_ptr());
  call("zmoe_lora_plan", dev, [&](zmoe_stream_t s) { return zmoe_lora_plan(ids, t, g, po, pt, s); });
  return py::make_tuple(offsets, tor);
}

// What lora and lora_grad have in common.
template <class A>
void adapters(A& args, const Tensor& a, const Tensor& b, const OptTensor& scale, const Tensor& offsets,
              const OptTensor& token_of_row, const OptTensor& rank, int64_t T, at::Device dev) {
  dims(a, "a", 3);
  dims(b, "b", 3);
  const int64_t G = a.size(0), R = a.size(1), H = a.size(2), N = b.size(1);
  args.a = arg<uint16_t>(a, "a", kBF16, {G, R, H}, dev);
  args.b = arg<uint16_t>(b, "b", kBF16, {G, N, R}, dev);
  args.scale = arg<float>(scale, "scale", kF32, {G}, dev);
  args.rank = arg<int32_t>(rank, "rank", kI32, {G}, dev);
  args.offsets = arg<int32_t>(offsets, "offsets", kI32, {G + 1}, dev);
  args.token_of_row = arg<int32_t>(token_of_row, "token_of_row", kI32, {T}, dev);
  args.T = to_int(T, "T");
  args.H = to_int(H, "H");
  args.N = to_int(N, "N");
  args.G = to_int(G, "G");
  args.R = to_int(R, "R");
}

Tensor lora(const Tensor& x, const OptTensor& base, const Tensor& a, const Tensor& b, const OptTensor& scale,
            const Tensor& offsets, const OptTensor& token_of_row, const OptTensor& rank, const OptTensor& out_,
            const OptTensor& u) {
  const at::Device dev = cuda(x, "x", 2);
  const int64_t T = x.size(0);
  zmoe_lora_args p{};
  adapters(p, a, b, scale, offsets, token_of_row, rank, T, dev);
  p.x = arg<uint16_t>(x, "x", kBF16, {T, (int64_t)p.H}, dev);
  p.base = arg<uint16_t>(base, "base", kBF16, {T, (int64_t)p.N}, dev);
  p.u = arg<float>(u, "u", kF32, {T, (int64_t)p.R}, dev);
  Tensor out = out_ ? *out_ : empty({T, (int64_t)p.N}, kBF16, dev), scratch;
  p.out = arg<uint16_t>(out, "out", kBF16, {T, (int64_t)p.N}, dev);
  if (T > ZMOE_LORA_ROWS) {
    scratch = empty({T, (int64_t)p.R}, kF32, dev);
    p.scratch = static_cast<float*>(scratch.data_ptr());
  }
  call("zmoe_lora", dev, [&](zmoe_stream_t s) { return zmoe_lora(&p, s); });
  return out;
}

py::tuple lora_grad(const Tensor& dy, const Tensor& x, const Tensor& u, const Tensor& a, const Tensor& b,
                    const OptTensor& scale, const Tensor& offsets, const OptTensor& token_of_row, const OptTensor& rank,
                    const OptTensor& base, const OptTensor& dx_) {
  const at::Device dev = cuda(dy, "dy", 2);
  const int64_t T = dy.size(0);
  zmoe_lora_grad_args p{};
  adapters(p, a, b, scale, offsets, token_of_row, rank, T, dev);
  p.dy = arg<uint16_t>(dy, "dy", kBF16, {T, (int64_t)p.N}, dev);
  p.x = arg<uint16_t>(x, "x", kBF16, {T, (int64_t)p.H}, dev);
  p.u = arg<float>(u, "u", kF32, {T, (int64_t)p.R}, dev);
  p.base = arg<uint16_t>(base, "base", kBF16, {T, (int64_t)p.H}, dev);
  Tensor dx = dx_ ? *dx_ : empty({T, (int64_t)p.H}, kBF16, dev);
  p.dx = arg<uint16_t>(dx, "dx", kBF16, {T, (int64_t)p.H}, dev);
  Tensor da = empty(a.sizes(), kBF16, dev), db = empty(b.sizes(), kBF16, dev),
         scratch = empty({T, (int64_t)p.R}, kF32, dev);
  p.da = static_cast<uint16_t*>(da.data_ptr());
  p.db = static_cast<uint16_t*>(db.data_ptr());
  p.scratch = static_cast<float*>(scratch.data_ptr());
  call("zmoe_lora_grad", dev, [&](zmoe_stream_t s) { return zmoe_lora_grad(&p, s); });
  return py::make_tuple(dx, da, db);
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
  g_error = new py::object(py::module_::import("zmoe._lib").attr("ZmoeError"));
  m.def("permute", &permute);
  m.def("permute_grad", &permute_grad);
  m.def("combine_grad", &combine_grad);
  m.def("lora_plan", &lora_plan);
  m.def("lora", &lora);
  m.def("lora_grad", &lora_grad);
}
