// The generation operators' calls from Python: argument checks, output and workspace allocation and the current
// stream, in C++, because a decode step's kernels are shorter than the same work done in Python (a call of
// linear_w4 for one row: 5 us of host time, as torch.add takes, instead of 20). Everything else is in the C ABI's entries, which these
// call. Module torch_xdna.lib._xdna_generate; generate.py documents the arguments.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <sstream>

#include "xdna_b200.h"

namespace {

PyObject *g_error = nullptr, *g_unavailable = nullptr;  // XdnaError, XdnaUnavailable

struct Raised {};  // a Python exception is set

[[noreturn]] void raise(const char* name, int status, const std::string& text) {
  PyObject* e = PyObject_CallFunction(g_error, "sis", name, status, text.c_str());
  if (e != nullptr) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

#define REQUIRE(cond, status, ...)            \
  do {                                        \
    if (!(cond)) {                            \
      std::ostringstream text_;               \
      text_ << __VA_ARGS__;                   \
      raise(name, status, text_.str());       \
    }                                         \
  } while (0)

const at::Tensor& tensor(const char* name, const char* what, PyObject* o) {
  REQUIRE(THPVariable_Check(o), XDNA_ERR_INVALID, what << ": not a tensor");
  return THPVariable_Unpack(o);
}

std::optional<at::Tensor> maybe(const char* name, const char* what, PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return tensor(name, what, o);
}

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return XDNA_F32;
    case at::kBFloat16: return XDNA_BF16;
    case at::kHalf: return XDNA_F16;
    default: return -1;
  }
}

const char* type(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return "float32";
    case at::kBFloat16: return "bfloat16";
    case at::kHalf: return "float16";
    default: return c10::toString(t.scalar_type());
  }
}

bool half(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
void* ptr(const std::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// t as the attention kernels read it: contiguous in the last dimension, every other stride a positive multiple of 8
// elements, 16-byte aligned; a copy where it is not. Strides of dimensions of at most one entry do not matter.
at::Tensor rows(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && aligned(t);
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t pitch_of(const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 8; }

// All tensors on the first one's GPU; that GPU current while the guard lives, and its current stream.
struct Place {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream = nullptr;
  Place(const char* name, const at::Tensor& first, std::initializer_list<const at::Tensor*> others) {
    if (!first.is_cuda()) {
      PyErr_SetString(g_unavailable, "torch_xdna ops run on CUDA tensors; move the model and inputs to the B200");
      throw Raised{};
    }
    for (const at::Tensor* t : others)
      REQUIRE(t == nullptr || t->device() == first.device(), XDNA_ERR_INVALID,
              "tensors on " << first.device() << " and " << t->device());
    guard.set_device(first.device());
    stream = c10::cuda::getCurrentCUDAStream(first.device().index()).stream();
  }
};

void check(const char* name, int rc) {
  if (rc != XDNA_OK) raise(name, rc, xdna_last_error());
}

const at::Tensor* in(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

// Whether autograd would record a call with these inputs. The call then returns None, and the custom op makes it: its
// result raises in backward, where one from here would have no history and the gradient would be missing without a word.
bool tracked(std::initializer_list<const at::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : inputs)
    if (t != nullptr && t->requires_grad()) return true;
  return false;
}

double scale_of(const char* name, const at::Tensor& q, const at::Tensor& kv, PyObject* scale) {
  const int64_t hq = q.size(1), d = q.size(2), hkv = kv.size(-2);
  REQUIRE(half(q), XDNA_ERR_INVALID, "bf16 or f16, not " << type(q));
  REQUIRE(hq >= 1 && hkv >= 1 && hq % hkv == 0 && hq / hkv <= 128, XDNA_ERR_INVALID,
          hq << " query heads do not share " << hkv << " key heads evenly (at most 128 each)");
  REQUIRE(d == 64 || d == 128, XDNA_ERR_UNSUPPORTED, "head dimension " << d << " (64 or 128)");
  if (scale == Py_None) return d == 64 ? 0.125 : 0.08838834764831845;
  const double s = PyFloat_AsDouble(scale);
  if (PyErr_Occurred()) throw Raised{};
  REQUIRE(s > 0 && s <= 2.3e38, XDNA_ERR_INVALID, "scale " << s << " is not positive and at most 2.3e38");
  return s;
}

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return n ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)) : at::Tensor();
}

at::Tensor packed_attention(PyObject* const* a) {
  const char* name = "packed_attention";
  const at::Tensor &q0 = tensor(name, "q", a[0]), &k0 = tensor(name, "k", a[1]), &v0 = tensor(name, "v", a[2]),
                   &cu = tensor(name, "cu_seqlens", a[3]);
  REQUIRE(q0.dim() == 3 && k0.dim() == 3 && k0.sizes() == v0.sizes() && k0.size(0) == q0.size(0) &&
              k0.size(2) == q0.size(2),
          XDNA_ERR_INVALID, "q " << q0.sizes() << ", k " << k0.sizes() << ", v " << v0.sizes()
                                 << ": need [T, Hq, D] and [T, Hkv, D]");
  REQUIRE(k0.scalar_type() == q0.scalar_type() && v0.scalar_type() == q0.scalar_type(), XDNA_ERR_INVALID,
          "q " << type(q0) << ", k " << type(k0) << ", v " << type(v0));
  REQUIRE(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.size(0) >= 1 && cu.is_contiguous(), XDNA_ERR_INVALID,
          "cu_seqlens: int32 [N + 1], contiguous");
  const double scale = scale_of(name, q0, k0, a[4]);
  if (tracked({&q0, &k0, &v0})) return {};
  Place place(name, q0, {&k0, &v0, &cu});
  const at::Tensor q = rows(q0), k = rows(k0), v = rows(v0);
  const int64_t T = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(1), n = cu.size(0) - 1;
  at::Tensor out = at::empty({T, hq, d}, q.options());
  const size_t size = xdna_packed_attention_workspace(n, T, hq, hkv);
  const at::Tensor ws = bytes(size, q);
  check(name, xdna_packed_attention(q.data_ptr(), pitch_of(q, 0), pitch_of(q, 1), k.data_ptr(), pitch_of(k, 0), pitch_of(k, 1),
                                    v.data_ptr(), pitch_of(v, 0), pitch_of(v, 1), cu.data_ptr<int32_t>(), n, T, hq, hkv, d,
                                    code(q.scalar_type()), static_cast<float>(scale), out.data_ptr(),
                                    size ? ws.data_ptr() : nullptr, size, place.stream));
  return out;
}

at::Tensor shared_prefix_attention(PyObject* const* a) {
  const char* name = "shared_prefix_attention";
  const at::Tensor &q0 = tensor(name, "q", a[0]), &pk0 = tensor(name, "prefix_k", a[1]),
                   &pv0 = tensor(name, "prefix_v", a[2]), &ck0 = tensor(name, "k_cache", a[3]),
                   &cv0 = tensor(name, "v_cache", a[4]), &lens = tensor(name, "cache_lens", a[5]);
  REQUIRE(q0.dim() == 3 && pk0.dim() == 3 && ck0.dim() == 4 && pk0.sizes() == pv0.sizes() && ck0.sizes() == cv0.sizes() &&
              ck0.size(0) == q0.size(0) && pk0.size(1) == ck0.size(2) && pk0.size(2) == ck0.size(3) &&
              pk0.size(2) == q0.size(2),
          XDNA_ERR_INVALID, "q " << q0.sizes() << ", prefix " << pk0.sizes() << " / " << pv0.sizes() << ", cache "
                                 << ck0.sizes() << " / " << cv0.sizes()
                                 << ": need [B, Hq, D], [P, Hkv, D] and [B, S, Hkv, D]");
  for (const at::Tensor* t : {&pk0, &pv0, &ck0, &cv0})
    REQUIRE(t->scalar_type() == q0.scalar_type(), XDNA_ERR_INVALID, "operands of several types");
  REQUIRE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == q0.size(0) && lens.is_contiguous(),
          XDNA_ERR_INVALID, "cache_lens: int32 [B], contiguous");
  const double scale = scale_of(name, q0, pk0, a[6]);
  if (tracked({&q0, &pk0, &pv0, &ck0, &cv0})) return {};
  Place place(name, q0, {&pk0, &pv0, &ck0, &cv0, &lens});
  const at::Tensor q = rows(q0), pk = rows(pk0), pv = rows(pv0), ck = rows(ck0), cv = rows(cv0);
  const int64_t B = q.size(0), hq = q.size(1), d = q.size(2), P = pk.size(0), hkv = pk.size(1), S = ck.size(1);
  at::Tensor out = at::empty({B, hq, d}, q.options());
  const size_t size = xdna_prefix_attention_workspace(B, P, S, hq, hkv, d);
  const at::Tensor ws = bytes(size, q);
  check(name, xdna_prefix_attention(
                  q.data_ptr(), pitch_of(q, 0), pitch_of(q, 1), pk.data_ptr(), pitch_of(pk, 0), pitch_of(pk, 1), pv.data_ptr(),
                  pitch_of(pv, 0), pitch_of(pv, 1), ck.data_ptr(), pitch_of(ck, 0), pitch_of(ck, 1), pitch_of(ck, 2),
                  cv.data_ptr(), pitch_of(cv, 0), pitch_of(cv, 1), pitch_of(cv, 2), lens.data_ptr<int32_t>(), B, P, S, hq,
                  hkv, d, code(q.scalar_type()), static_cast<float>(scale), out.data_ptr(),
                  size ? ws.data_ptr() : nullptr, size, place.stream));
  return out;
}

at::Tensor linear_w4(PyObject* const* a) {
  const char* name = "linear_w4";
  const at::Tensor &x = tensor(name, "x", a[0]), &codes = tensor(name, "codes", a[1]),
                   &scales = tensor(name, "scales", a[2]);
  const int64_t group = PyLong_AsLongLong(a[3]);
  if (group == -1 && PyErr_Occurred()) throw Raised{};
  std::optional<at::Tensor> bias = maybe(name, "bias", a[4]);
  REQUIRE(x.dim() >= 1 && code(x.scalar_type()) >= 0, XDNA_ERR_INVALID,
          "x " << x.sizes() << " " << type(x) << ": f32, bf16 or f16");
  const int64_t K = x.size(-1), half_row = (K + 127) / 128 * 64;
  REQUIRE(group == 32 || group == 64 || group == 128, XDNA_ERR_INVALID, "group " << group << " (32, 64 or 128)");
  REQUIRE(codes.dim() == 2 && codes.scalar_type() == at::kByte && codes.is_contiguous() && aligned(codes) && K >= 1 &&
              codes.size(1) == half_row,
          XDNA_ERR_INVALID, "codes " << codes.sizes() << " " << type(codes) << " for K = " << K
                                     << ": need contiguous, aligned uint8 [N, " << half_row << "]");
  const int64_t N = codes.size(0), groups = (K + group - 1) / group;
  REQUIRE(scales.dim() == 2 && scales.size(0) == N && scales.size(1) == groups && half(scales) && scales.is_contiguous(),
          XDNA_ERR_INVALID, "scales " << scales.sizes() << " " << type(scales)
                                      << ": need contiguous bf16 or f16 [" << N << ", " << groups << "]");
  REQUIRE(!bias || (bias->dim() == 1 && bias->size(0) == N && code(bias->scalar_type()) >= 0), XDNA_ERR_INVALID,
          "bias: [N] in f32, bf16 or f16");
  if (tracked({&x, &scales, in(bias)})) return {};
  Place place(name, x, {&codes, &scales, in(bias)});
  const at::Tensor sc = reinterpret_cast<uintptr_t>(scales.data_ptr()) % 4 ? scales.clone() : scales;
  at::Tensor x2 = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  const int64_t M = x2.size(0);
  if (x2.stride(1) != 1 || (M > 1 && x2.stride(0) < K)) x2 = x2.clone(at::MemoryFormat::Contiguous);
  if (bias && !bias->is_contiguous()) bias = bias->contiguous();
  at::Tensor y = at::empty({M, N}, x.options());
  check(name, xdna_linear_w4(x2.data_ptr(), code(x.scalar_type()), M, K, M > 1 ? x2.stride(0) : K,
                             codes.data_ptr<uint8_t>(), sc.data_ptr(), code(scales.scalar_type()),
                             static_cast<int>(group), N, ptr(bias), bias ? code(bias->scalar_type()) : XDNA_F32,
                             y.data_ptr(), N, place.stream));
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  return y.view(shape);
}

at::Tensor process_logits(PyObject* const* a) {
  const char* name = "process_logits";
  at::Tensor logits = tensor(name, "logits", a[0]);
  std::optional<at::Tensor> tokens = maybe(name, "tokens", a[1]);
  static const char* const kRow[] = {"lens", "prompt_lens", "repetition", "presence", "frequency"};
  std::optional<at::Tensor> row[5], bias = maybe(name, "bias", a[7]), mask = maybe(name, "mask", a[8]);
  REQUIRE(logits.dim() == 2 && code(logits.scalar_type()) >= 0, XDNA_ERR_INVALID,
          "logits " << logits.sizes() << " " << type(logits) << ": [B, V] in f32, bf16 or f16");
  const int64_t B = logits.size(0), V = logits.size(1), words = (V + 31) / 32;
  if (tokens)
    REQUIRE(tokens->dim() == 2 && tokens->size(0) == B &&
                (tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong),
            XDNA_ERR_INVALID, "tokens " << tokens->sizes() << " " << type(*tokens) << ": int32 or int64 [B, T]");
  for (int i = 0; i < 5; ++i) {
    row[i] = maybe(name, kRow[i], a[2 + i]);
    if (!row[i]) continue;
    REQUIRE(tokens, XDNA_ERR_INVALID, kRow[i] << " without tokens");
    REQUIRE(row[i]->dim() == 1 && row[i]->size(0) == B && row[i]->scalar_type() == (i < 2 ? at::kInt : at::kFloat) &&
                row[i]->is_contiguous(),
            XDNA_ERR_INVALID, kRow[i] << ": contiguous " << (i < 2 ? "int32" : "float32") << " [B]");
  }
  if (bias)
    REQUIRE(bias->scalar_type() == at::kFloat &&
                ((bias->dim() == 1 && bias->size(0) == V) ||
                 (bias->dim() == 2 && bias->size(1) == V && (bias->size(0) == B || bias->size(0) == 1))),
            XDNA_ERR_INVALID, "bias: f32 [V] or [B, V]");
  if (mask)
    REQUIRE(mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(1) == words &&
                (mask->size(0) == B || mask->size(0) == 1),
            XDNA_ERR_INVALID, "mask: int32 [B, " << words << "] or [1, " << words << "]");
  if (tracked({&logits, in(row[2]), in(row[3]), in(row[4]), in(bias)})) return {};
  Place place(name, logits, {in(tokens), in(row[0]), in(row[1]), in(row[2]), in(row[3]), in(row[4]), in(bias), in(mask)});
  // rows contiguous
  for (at::Tensor* t : {&logits, tokens ? &*tokens : nullptr, bias ? &*bias : nullptr, mask ? &*mask : nullptr})
    if (t != nullptr && t->size(-1) > 1 && t->stride(-1) != 1) *t = t->contiguous();
  auto pitch = [](const std::optional<at::Tensor>& t) { return t && t->dim() == 2 && t->size(0) > 1 ? t->stride(0) : 0; };
  at::Tensor out = at::empty({B, V}, logits.options());
  check(name, xdna_process_logits(
                  logits.data_ptr(), code(logits.scalar_type()), B, V, B > 1 ? logits.stride(0) : V, ptr(tokens),
                  tokens && tokens->scalar_type() == at::kLong ? 8 : 4, tokens ? tokens->size(1) : 0, pitch(tokens),
                  static_cast<const int32_t*>(ptr(row[0])), static_cast<const int32_t*>(ptr(row[1])),
                  static_cast<const float*>(ptr(row[2])), static_cast<const float*>(ptr(row[3])),
                  static_cast<const float*>(ptr(row[4])), static_cast<const float*>(ptr(bias)), pitch(bias),
                  static_cast<const uint32_t*>(ptr(mask)), pitch(mask), out.data_ptr(), V, place.stream));
  return out;
}

thread_local int64_t t_launches = 0;  // kernels of the last call

template <at::Tensor (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", N, n);
    return nullptr;
  }
  try {
    const int64_t before = xdna_launch_count();
    at::Tensor out = F(args);
    t_launches = xdna_launch_count() - before;
    return THPVariable_Wrap(std::move(out));
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* launches(PyObject*, PyObject*) { return PyLong_FromLongLong(t_launches); }

PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "XdnaError, XdnaUnavailable");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  g_error = args[0];
  g_unavailable = args[1];
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef kMethods[] = {
    {"init", FAST(init), METH_FASTCALL, "the exception types"},
    {"launches", launches, METH_NOARGS, "kernels that this thread's last call enqueued"},
    {"packed_attention", FAST((call<packed_attention, 5>)), METH_FASTCALL, nullptr},
    {"shared_prefix_attention", FAST((call<shared_prefix_attention, 7>)), METH_FASTCALL, nullptr},
    {"linear_w4", FAST((call<linear_w4, 5>)), METH_FASTCALL, nullptr},
    {"process_logits", FAST((call<process_logits, 9>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_xdna_generate", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__xdna_generate() { return PyModule_Create(&kModule); }
