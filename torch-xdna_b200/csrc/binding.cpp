// The generation operators' calls from Python: argument checks, output and workspace allocation and the current
// stream, in C++, because a decode step's kernels are shorter than the same work done in Python (a call of
// linear_w4 for one row: 5 us of host time, as torch.add takes, instead of 20). Everything else is in the C ABI's entries, which these
// call. Module torch_xdna.lib._xdna_generate; generate.py and layer.py document the arguments.
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

// Says to autograd that t has been written in place, so that backward notices where it was saved before. (Tensors of
// inference mode keep no such count.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

double scale_of(const char* name, const at::Tensor& q, int64_t hq, int64_t hkv, int64_t d, PyObject* scale) {
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

double scale_of(const char* name, const at::Tensor& q, const at::Tensor& kv, PyObject* scale) {
  return scale_of(name, q, q.size(1), kv.size(-2), q.size(2), scale);
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

// ---------------------------------------------------------------- a decoder layer around its products (layer.py)
double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Raised{};
  return x;
}

bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw Raised{};
  return x != 0;
}

float eps_of(const char* name, PyObject* o) {
  const double eps = number(o);
  REQUIRE(eps >= 0 && eps <= 3e38, XDNA_ERR_INVALID, "eps " << eps);
  return static_cast<float>(eps);
}

float factor_of(const char* name, const char* what, PyObject* o) {
  const double x = number(o);
  REQUIRE(x >= -3e38 && x <= 3e38, XDNA_ERR_INVALID, what << " " << x);
  return static_cast<float>(x);
}

// A head's frequencies: f32 [R / 2], R at most D.
void check_freq(const char* name, const std::optional<at::Tensor>& f, int64_t d) {
  REQUIRE(!f || (f->dim() == 1 && f->scalar_type() == at::kFloat && f->is_contiguous() && 2 * f->size(0) <= d), XDNA_ERR_INVALID,
          "inv_freq: contiguous float32 [R / 2], R at most " << d);
}

// A norm's weights: [D], or [H, D] with one row per head.
void check_norm(const char* name, const char* what, const std::optional<at::Tensor>& w, int64_t h, int64_t d) {
  REQUIRE(!w || (code(w->scalar_type()) >= 0 && (w->dim() == 1 || (w->dim() == 2 && w->size(0) == h)) && w->size(-1) == d), XDNA_ERR_INVALID,
          what << ": [" << d << "] or [" << h << ", " << d << "] in f32, bf16 or f16");
}

// Contiguous and aligned, a copy where it is not.
void settle(std::optional<at::Tensor>& t) {
  if (t && !(t->is_contiguous() && aligned(*t))) t = t->clone(at::MemoryFormat::Contiguous);
}
int64_t per_head(const std::optional<at::Tensor>& w) { return w && w->dim() == 2 ? w->size(1) : 0; }
int dtype_of(const std::optional<at::Tensor>& t) { return t ? code(t->scalar_type()) : XDNA_F32; }

at::Tensor rotary(PyObject* const* a) {
  const char* name = "rotary";
  const at::Tensor &x0 = tensor(name, "x", a[0]), &pos = tensor(name, "positions", a[1]);
  const std::optional<at::Tensor> freq = tensor(name, "inv_freq", a[2]);
  std::optional<at::Tensor> norm = maybe(name, "norm", a[5]);
  const float factor = factor_of(name, "factor", a[3]), eps = eps_of(name, a[6]);
  const bool interleaved = truth(a[4]);
  REQUIRE(x0.dim() == 3 && code(x0.scalar_type()) >= 0, XDNA_ERR_INVALID,
          "x " << x0.sizes() << " " << type(x0) << ": [T, H, D] in f32, bf16 or f16");
  const int64_t T = x0.size(0), H = x0.size(1), D = x0.size(2);
  REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, XDNA_ERR_UNSUPPORTED, "head dimension " << D << " (multiples of 8 up to 256)");
  REQUIRE(pos.dim() == 1 && pos.size(0) == T && pos.is_contiguous() && (pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong),
          XDNA_ERR_INVALID, "positions: contiguous int32 or int64 [" << T << "]");
  check_freq(name, freq, D);
  check_norm(name, "norm", norm, H, D);
  if (tracked({&x0, in(freq), in(norm)})) return {};
  Place place(name, x0, {&pos, in(freq), in(norm)});
  const at::Tensor x = rows(x0);
  settle(norm);
  at::Tensor out = at::empty({T, H, D}, x.options());
  check(name, xdna_rotary(x.data_ptr(), code(x.scalar_type()), T, H, D, pitch_of(x, 0), pitch_of(x, 1), pos.data_ptr(),
                          pos.scalar_type() == at::kLong ? 8 : 4, static_cast<const float*>(ptr(freq)), freq->size(0), factor,
                          interleaved, ptr(norm), dtype_of(norm), per_head(norm), eps, out.data_ptr(), place.stream));
  return out;
}

struct Two {
  at::Tensor first, second;  // undefined where autograd would record the call
};

Two add_norm(PyObject* const* a) {
  const char* name = "add_norm";
  const at::Tensor &x = tensor(name, "x", a[0]), &y = tensor(name, "y", a[1]);
  std::optional<at::Tensor> w = tensor(name, "weight", a[2]), post = maybe(name, "post", a[3]), gate = maybe(name, "gate", a[4]);
  const float scale = factor_of(name, "scale", a[5]), eps = eps_of(name, a[6]);
  REQUIRE(x.dim() >= 1 && x.sizes() == y.sizes() && code(x.scalar_type()) >= 0 && code(y.scalar_type()) >= 0, XDNA_ERR_INVALID,
          "x " << x.sizes() << " " << type(x) << ", y " << y.sizes() << " " << type(y) << ": one shape [..., D], f32, bf16 or f16");
  const int64_t D = x.size(-1);
  REQUIRE(D >= 1 && D <= 16384, XDNA_ERR_UNSUPPORTED, "rows of " << D << " entries (1 to 16384)");
  for (const auto& v : {std::make_pair("weight", &w), std::make_pair("post", &post)})
    REQUIRE(!*v.second || ((*v.second)->dim() == 1 && (*v.second)->size(0) == D && code((*v.second)->scalar_type()) >= 0), XDNA_ERR_INVALID,
            v.first << ": [" << D << "] in f32, bf16 or f16");
  REQUIRE(!gate || (code(gate->scalar_type()) >= 0 && (gate->sizes() == x.sizes() || (gate->dim() == 1 && gate->size(0) == D))),
          XDNA_ERR_INVALID, "gate: [" << D << "] or x's shape, in f32, bf16 or f16");
  if (tracked({&x, &y, in(w), in(post), in(gate)})) return {};
  Place place(name, x, {&y, in(w), in(post), in(gate)});
  const int64_t n = x.numel() / D;
  // as rows: [n, D] with entries side by side
  auto flat = [&](const at::Tensor& t) {
    at::Tensor r = t.dim() == 2 ? t : t.reshape({n, D});
    return r.stride(1) != 1 && D > 1 ? r.contiguous() : r;
  };
  auto pitch = [&](const at::Tensor& t) { return n > 1 ? t.stride(0) : D; };
  const at::Tensor x2 = flat(x), y2 = flat(y);
  settle(w);
  settle(post);
  const bool each = gate && !(gate->dim() == 1 && (x.dim() > 1 || n == 1));
  if (each) gate = flat(*gate);
  if (gate && !each) settle(gate);
  Two out{at::empty(x.sizes(), x.options()), at::empty(y.sizes(), y.options())};
  check(name, xdna_add_norm(x2.data_ptr(), code(x.scalar_type()), pitch(x2), y2.data_ptr(), code(y.scalar_type()), pitch(y2), n, D, ptr(w),
                            dtype_of(w), ptr(post), dtype_of(post), ptr(gate), dtype_of(gate), each ? pitch(*gate) : 0, scale, eps,
                            out.first.data_ptr(), out.second.data_ptr(), place.stream));
  return out;
}

// The four tensors of a paged cache: codes [pages, Hkv, page, D], scales [pages, Hkv].
struct Cache {
  const at::Tensor &k, &v, &ks, &vs;
  int64_t pages, hkv, page, d;
  Cache(const char* name, PyObject* const* a)
      : k(tensor(name, "k_cache", a[0])), v(tensor(name, "v_cache", a[1])), ks(tensor(name, "k_scales", a[2])), vs(tensor(name, "v_scales", a[3])) {
    REQUIRE(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() &&
                (k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn),
            XDNA_ERR_INVALID, "caches " << k.sizes() << " " << type(k) << " / " << v.sizes() << " " << type(v)
                                        << ": need [pages, Hkv, page, D] in int8 or float8_e4m3fn");
    pages = k.size(0), hkv = k.size(1), page = k.size(2), d = k.size(3);
    REQUIRE(d == 64 || d == 128, XDNA_ERR_UNSUPPORTED, "head dimension " << d << " (64 or 128)");
    REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, XDNA_ERR_UNSUPPORTED, "pages of " << page << " tokens (16, 32, 64 or 128)");
    REQUIRE(hkv >= 1, XDNA_ERR_INVALID, "no key heads");
    for (const at::Tensor* t : {&k, &v})
      REQUIRE(t->stride(3) == 1 && t->stride(2) == d && (hkv == 1 || t->stride(1) == page * d) &&
                  (pages <= 1 || (t->stride(0) >= hkv * page * d && t->stride(0) % 16 == 0)) && aligned(*t),
              XDNA_ERR_INVALID, "caches: a page's [Hkv, page, D] contiguous and aligned to 16 bytes, pages apart");
    for (const at::Tensor* t : {&ks, &vs})
      REQUIRE(t->dim() == 2 && t->size(0) == pages && t->size(1) == hkv && t->scalar_type() == at::kFloat && (hkv == 1 || t->stride(1) == 1) &&
                  (pages <= 1 || t->stride(0) >= hkv),
              XDNA_ERR_INVALID, "scales: float32 [" << pages << ", " << hkv << "], a page's contiguous");
  }
  int format() const { return k.scalar_type() == at::kChar ? XDNA_I8 : XDNA_E4M3; }
  int64_t pitch(const at::Tensor& t) const { return pages > 1 ? t.stride(0) : 0; }
};

const at::Tensor& table_of(const char* name, PyObject* o, int64_t n) {
  const at::Tensor& t = tensor(name, "table", o);
  REQUIRE(t.dim() == 2 && t.size(0) == n && t.scalar_type() == at::kInt && (t.size(1) <= 1 || t.stride(1) == 1) &&
              (n <= 1 || t.stride(0) >= 0),
          XDNA_ERR_INVALID, "table: int32 [" << n << ", pages of a sequence], rows contiguous");
  return t;
}

const at::Tensor& counts_of(const char* name, const char* what, PyObject* o, int64_t n) {
  const at::Tensor& t = tensor(name, what, o);
  REQUIRE(t.dim() == 1 && (n < 0 || t.size(0) == n) && t.scalar_type() == at::kInt && t.is_contiguous(), XDNA_ERR_INVALID,
          what << ": contiguous int32" << (n < 0 ? "" : ", one for each sequence"));
  return t;
}

// False without queries, None where autograd would record the call, else the queries.
PyObject* cache_append(PyObject* const* a) {
  const char* name = "cache_append";
  const at::Tensor &k0 = tensor(name, "k", a[0]), &v0 = tensor(name, "v", a[1]);
  const Cache c(name, a + 2);
  const std::optional<at::Tensor> cu = maybe(name, "cu_seqlens", a[8]), freq = maybe(name, "inv_freq", a[9]), q0 = maybe(name, "q", a[13]);
  std::optional<at::Tensor> k_norm = maybe(name, "k_norm", a[12]), q_norm = maybe(name, "q_norm", a[14]);
  const float factor = factor_of(name, "factor", a[10]), eps = eps_of(name, a[15]);
  const bool interleaved = truth(a[11]);
  REQUIRE(k0.dim() == 3 && k0.sizes() == v0.sizes() && k0.size(1) == c.hkv && k0.size(2) == c.d && half(k0) && v0.scalar_type() == k0.scalar_type(),
          XDNA_ERR_INVALID, "k " << k0.sizes() << " " << type(k0) << ", v " << v0.sizes() << " " << type(v0) << ": need [T, " << c.hkv << ", " << c.d
                                 << "] in bf16 or f16");
  const int64_t T = k0.size(0);
  REQUIRE(!q0 || (q0->dim() == 3 && q0->size(0) == T && q0->size(1) >= 1 && q0->size(2) == c.d && q0->scalar_type() == k0.scalar_type()),
          XDNA_ERR_INVALID, "q: [" << T << ", Hq, " << c.d << "] in k's type");
  if (cu) counts_of(name, "cu_seqlens", a[8], -1);
  REQUIRE(!cu || cu->size(0) >= 1, XDNA_ERR_INVALID, "cu_seqlens: contiguous int32 [N + 1]");
  const int64_t n = cu ? cu->size(0) - 1 : T;
  const at::Tensor &table = table_of(name, a[6], n), &starts = counts_of(name, "starts", a[7], n);
  check_freq(name, freq, c.d);
  check_norm(name, "k_norm", k_norm, c.hkv, c.d);
  REQUIRE(q0 || !q_norm, XDNA_ERR_INVALID, "q_norm without q");
  if (q0) check_norm(name, "q_norm", q_norm, q0->size(1), c.d);
  REQUIRE(!tracked({&k0, &v0, in(k_norm), &c.k, &c.v, &c.ks, &c.vs}), XDNA_ERR_INVALID,
          "a cache keeps no gradients: keys and values that require grad, and into a cache that does, are stored under torch.no_grad()");
  if (tracked({in(q0), in(q_norm), in(freq)})) Py_RETURN_NONE;
  Place place(name, k0, {&v0, &c.k, &c.v, &c.ks, &c.vs, &table, &starts, in(cu), in(freq), in(q0), in(k_norm), in(q_norm)});
  const at::Tensor k = rows(k0), v = rows(v0);
  const at::Tensor q = q0 ? rows(*q0) : at::Tensor();
  settle(k_norm);
  settle(q_norm);
  const int64_t hq = q0 ? q.size(1) : 0;
  at::Tensor out = q0 ? at::empty({T, hq, c.d}, q.options()) : at::Tensor();
  check(name, xdna_cache_append(
                  k.data_ptr(), pitch_of(k, 0), pitch_of(k, 1), v.data_ptr(), pitch_of(v, 0), pitch_of(v, 1), code(k.scalar_type()), T, c.hkv, c.d,
                  c.k.data_ptr(), c.pitch(c.k), c.v.data_ptr(), c.pitch(c.v), c.format(), c.ks.data_ptr<float>(), c.pitch(c.ks),
                  c.vs.data_ptr<float>(), c.pitch(c.vs), c.pages, c.page, table.data_ptr<int32_t>(), n > 1 ? table.stride(0) : 0, table.size(1),
                  starts.data_ptr<int32_t>(), static_cast<const int32_t*>(ptr(cu)), n, static_cast<const float*>(ptr(freq)),
                  freq ? freq->size(0) : 0, factor, interleaved, ptr(k_norm), dtype_of(k_norm), per_head(k_norm), eps,
                  q0 ? q.data_ptr() : nullptr, q0 ? pitch_of(q, 0) : 8, q0 ? pitch_of(q, 1) : 8, hq, ptr(q_norm), dtype_of(q_norm),
                  per_head(q_norm), q0 ? out.data_ptr() : nullptr, place.stream));
  for (const at::Tensor* t : {&c.k, &c.v, &c.ks, &c.vs}) written(*t);
  if (!q0) Py_RETURN_FALSE;
  return THPVariable_Wrap(std::move(out));
}

at::Tensor paged_attention(PyObject* const* a) {
  const char* name = "paged_attention";
  const at::Tensor& q0 = tensor(name, "q", a[0]);
  const Cache c(name, a + 1);
  REQUIRE((q0.dim() == 3 || q0.dim() == 4) && q0.size(-1) == c.d, XDNA_ERR_INVALID,
          "q " << q0.sizes() << ": need [B, Hq, " << c.d << "] or [B, T, Hq, " << c.d << "]");
  const at::Tensor q4 = q0.dim() == 4 ? q0 : q0.unsqueeze(1);
  const int64_t B = q4.size(0), T = q4.size(1), hq = q4.size(2);
  const double scale = scale_of(name, q4, hq, c.hkv, c.d, a[7]);
  const at::Tensor &table = table_of(name, a[5], B), &lens = counts_of(name, "lens", a[6], B);
  if (tracked({&q0, &c.k, &c.v, &c.ks, &c.vs})) return {};
  Place place(name, q0, {&c.k, &c.v, &c.ks, &c.vs, &table, &lens});
  const at::Tensor q = rows(q4);
  at::Tensor out = at::empty(q0.sizes(), q0.options());
  const size_t size = xdna_paged_attention_workspace(B, T, hq, c.hkv, c.d, table.size(1) * c.page);
  const at::Tensor ws = bytes(size, q);
  check(name, xdna_paged_attention(q.data_ptr(), pitch_of(q, 0), pitch_of(q, 1), pitch_of(q, 2), code(q.scalar_type()), B, T, hq, c.hkv, c.d,
                                   c.k.data_ptr(), c.pitch(c.k), c.v.data_ptr(), c.pitch(c.v), c.format(), c.ks.data_ptr<float>(), c.pitch(c.ks),
                                   c.vs.data_ptr<float>(), c.pitch(c.vs), c.pages, c.page, table.data_ptr<int32_t>(),
                                   B > 1 ? table.stride(0) : 0, table.size(1), lens.data_ptr<int32_t>(), static_cast<float>(scale),
                                   out.data_ptr(), size ? ws.data_ptr() : nullptr, size, place.stream));
  return out;
}

thread_local int64_t t_launches = 0;  // kernels of the last call

PyObject* wrap(at::Tensor&& t) { return THPVariable_Wrap(std::move(t)); }
PyObject* wrap(Two&& t) {
  if (!t.first.defined()) Py_RETURN_NONE;
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(t.first)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(t.second)));
  return pair;
}
PyObject* wrap(PyObject* o) { return o; }

template <auto F, int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", N, n);
    return nullptr;
  }
  try {
    const int64_t before = xdna_launch_count();
    auto out = F(args);
    t_launches = xdna_launch_count() - before;
    return wrap(std::move(out));
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
    {"rotary", FAST((call<rotary, 7>)), METH_FASTCALL, nullptr},
    {"add_norm", FAST((call<add_norm, 7>)), METH_FASTCALL, nullptr},
    {"cache_append", FAST((call<cache_append, 16>)), METH_FASTCALL, nullptr},
    {"paged_attention", FAST((call<paged_attention, 8>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_xdna_generate", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__xdna_generate() { return PyModule_Create(&kModule); }
