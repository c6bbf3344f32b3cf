// torch_binding.cpp — CPython module that takes torch tensors straight to the C ABI for the
// operators a decode step calls once per layer (rope_kv_append, rope_kv_append_int4,
// kv_gather_int4, paged_decode_attention_int4, prompt_attention, shared_prefix_decode_attention,
// cross_attention_packed, sample_rows).
//
// Their kernels take a few microseconds, while checking some fifteen tensors from Python and
// converting thirty arguments through ctypes took 8 to 11 (append of a 64-request step: 14.7 us
// a call, of which the launch 3.1).  Here the same checks read the tensors directly.  The module
// holds no kernel and no state but the workspaces of calls that bring none: setup()
// is given the addresses of the C ABI's functions, so it serves whichever libspd_b200.so the
// process has loaded.  Every refusal is a Python RuntimeError; no C++ exception leaves it.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/DynamicTypes.h>

#include <algorithm>
#include <array>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "spd_b200.h"

namespace {

decltype(&spd_rope_kv_append) f_rope_append;
decltype(&spd_rope_kv_append_int4) f_rope_append_int4;
decltype(&spd_kv_gather_int4) f_gather;
decltype(&spd_paged_decode_attn_int4_err) f_decode;
decltype(&spd_paged_decode_attn_int4_workspace_size) f_decode_size;
decltype(&spd_prompt_attn) f_prompt;
decltype(&spd_kv_int4_page_bytes) f_page_bytes;
decltype(&spd_get_last_error) f_last_error;
decltype(&spd_stream_capture_id) f_capture_id;
decltype(&spd_shared_prefix_attn) f_prefix;
decltype(&spd_shared_prefix_attn_workspace_size) f_prefix_size;
decltype(&spd_sample_rows) f_sample;
decltype(&spd_cross_attn_packed) f_cross;
decltype(&spd_cross_attn_packed_workspace_size) f_cross_size;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void refuse(const char* name, const A&... parts) {
  std::ostringstream s;
  s << name << ": ";
  (s << ... << parts);
  throw Refused(s.str());
}

std::string shape_of(const at::Tensor& t) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << ")";
  return s.str();
}

// A tensor argument, or an undefined tensor for None where `optional`.
const at::Tensor& tensor(const char* name, const char* what, PyObject* o, bool optional = false) {
  static const at::Tensor* none = new at::Tensor();
  if (optional && o == Py_None) return *none;
  if (!THPVariable_Check(o)) refuse(name, what, " must be a tensor");
  return THPVariable_Unpack(o);
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int dtype_code(const char* name, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPD_F32;
    case at::kHalf: return SPD_F16;
    case at::kBFloat16: return SPD_BF16;
    default: refuse(name, "dtype ", c10::toString(t), " is not supported (float32/float16/bfloat16)");
  }
}

// All on the current CUDA device, whose current stream is launched on.
int current_device(const char* name, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t->defined() && !t->is_cuda()) refuse(name, "CUDA tensors required (the B200 kernels have no CPU fallback)");
  const int dev = (int)c10::cuda::current_device();
  for (const at::Tensor* t : ts)
    if (t->defined() && t->get_device() != dev) refuse(name, "all tensors must be on the current CUDA device");
  return dev;
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

int small_int(const char* name, const char* what, int64_t v) {
  if (v < 0 || v > INT32_MAX) refuse(name, what, " ", v, " is out of range");
  return (int)v;
}

void int32_vector(const char* name, const char* what, const at::Tensor& t, int64_t n) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse(name, what, " must be a contiguous int32 [", n, "] tensor");
}

int table_columns(const char* name, const at::Tensor& t, int64_t B) {
  if (t.dim() != 2 || t.size(0) != B || t.scalar_type() != at::kInt || !t.is_contiguous())
    refuse(name, "block_tables must be contiguous int32 [B, max_blocks]");
  return small_int(name, "max_blocks", t.size(1));
}

// Token and head strides of [n, H, D] with contiguous D; those of a dimension of one entry,
// which nothing steps over, are taken as dense.
std::pair<int64_t, int64_t> token_strides(const char* name, const char* what, const at::Tensor& t) {
  if (t.stride(2) != 1 && t.size(2) > 1) refuse(name, what, " needs a contiguous last dimension");
  const int64_t sh = t.size(1) == 1 ? t.size(2) : t.stride(1);
  return {t.size(0) > 1 ? t.stride(0) : sh * t.size(1), sh};
}

bool overlap(const at::Tensor& a, const at::Tensor& b) {
  auto span = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const char* p = static_cast<const char*>(t.const_data_ptr());
    return std::pair<const char*, const char*>(p, p + (last + 1) * t.element_size());
  };
  if (!a.numel() || !b.numel()) return false;
  const auto x = span(a), y = span(b);
  return x.first < y.second && y.first < x.second;
}

// `out` (contiguous, of q's shape) over some of q, but not over each of its elements in its place
bool partly_over(const at::Tensor& q, const at::Tensor& out) {
  return overlap(q, out) && !(q.const_data_ptr() == out.const_data_ptr() && q.is_contiguous());
}

void error_word(const char* name, const at::Tensor& t) {
  if (t.defined() && (t.scalar_type() != at::kInt || t.numel() < 1)) refuse(name, "error_word must be an int32 tensor");
}

int int4_block_size(const char* name, const at::Tensor& pool, int64_t Hkv, int64_t D) {
  if (pool.scalar_type() != at::kByte || pool.dim() != 3 || pool.size(1) != Hkv || !pool.is_contiguous())
    refuse(name, "pool must be a contiguous uint8 [num_blocks, ", Hkv, ", page bytes] tensor");
  for (int bs : {8, 16, 32})
    if (D <= INT32_MAX && (int64_t)f_page_bytes((int)D, bs) == pool.size(2) && pool.size(2) > 0) return bs;
  refuse(name, "pages of ", pool.size(2), " bytes fit no block size at head_dim ", D);
}

void check(int rc, const char* name) {
  if (rc == SPD_OK) return;
  char text[512] = {0};
  f_last_error(text, sizeof(text));
  std::ostringstream s;
  s << "spd_" << name << " failed (status " << rc << "): " << text;
  throw Refused(s.str());
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused("a truth value was expected");
  return v != 0;
}

void count(const char* name, Py_ssize_t given, Py_ssize_t wanted) {
  if (given != wanted) refuse(name, wanted, " arguments expected, ", given, " given");
}

// (q, k, v, cos, sin, k_pool, v_pool, block_tables, positions, cu_seqlens, interleaved, q_out, error_word);
// v_pool is None for the 4-bit form.
at::Tensor rope_append(const char* name, bool int4, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 13);
  const at::Tensor &q = tensor(name, "q", a[0], true), &k = tensor(name, "k", a[1]), &v = tensor(name, "v", a[2]),
                   &cos = tensor(name, "cos", a[3]), &sin = tensor(name, "sin", a[4]), &pool = tensor(name, "pool", a[5]),
                   &v_pool = tensor(name, "v_pool", a[6], int4), &tables = tensor(name, "block_tables", a[7]),
                   &positions = tensor(name, "positions", a[8]), &cu = tensor(name, "cu_seqlens", a[9], true),
                   &given = tensor(name, "q_out", a[11], true), &err = tensor(name, "error_word", a[12], true);
  current_device(name, {&k, &q, &v, &cos, &sin, &pool, &v_pool, &tables, &positions, &cu, &given, &err});
  if (k.dim() != 3 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
    refuse(name, "k and v must be [N, Hkv, D] of one shape and dtype");
  const int N = small_int(name, "N", k.size(0)), Hkv = small_int(name, "Hkv", k.size(1)), D = small_int(name, "D", k.size(2));
  int bs;
  if (int4) {
    bs = int4_block_size(name, pool, Hkv, D);
  } else {
    for (const at::Tensor* p : {&pool, &v_pool})
      if (p->dim() != 4 || p->size(2) != Hkv || p->size(3) != D || p->sizes() != pool.sizes() ||
          p->scalar_type() != k.scalar_type() || !p->is_contiguous())
        refuse(name, "pools must be contiguous [num_blocks, block_size, Hkv, D] of k's dtype");
    bs = small_int(name, "block_size", pool.size(1));
  }
  const int64_t B = positions.dim() == 1 ? positions.size(0) : -1;
  int32_vector(name, "positions", positions, B);
  const int max_blocks = table_columns(name, tables, B);
  if (cu.defined()) int32_vector(name, "cu_seqlens", cu, B + 1);
  else if (N != B)
    refuse(name, "without cu_seqlens one token per sequence is expected (", N, " tokens, ", B, " sequences)");
  if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || sin.sizes() != cos.sizes() ||
      !cos.is_contiguous() || !sin.is_contiguous())
    refuse(name, "cos and sin must be contiguous float32 [positions, rotated / 2] tables");
  const auto ks = token_strides(name, "k", k), vs = token_strides(name, "v", v);
  std::pair<int64_t, int64_t> qs{0, 0};
  int Hq = 0;
  at::Tensor out;
  if (q.defined()) {
    if (q.dim() != 3 || q.size(0) != N || q.size(2) != D || q.scalar_type() != k.scalar_type())
      refuse(name, "q ", shape_of(q), " does not match k ", shape_of(k));
    Hq = small_int(name, "Hq", q.size(1));
    qs = token_strides(name, "q", q);
    if (!given.defined()) out = at::empty(q.sizes(), q.options());
    else if (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !given.is_contiguous() ||
             overlap(q, given) || overlap(k, given) || overlap(v, given))
      refuse(name, "q_out must be a contiguous ", shape_of(q), " tensor of q's dtype apart from q, k and v");
    else out = given;
  } else if (given.defined()) {
    refuse(name, "q_out without q");
  }
  error_word(name, err);
  const int code = dtype_code(name, k.scalar_type()), rot = small_int(name, "rotated", 2 * cos.size(1)),
            max_pos = small_int(name, "positions", cos.size(0)), blocks = small_int(name, "num_blocks", pool.size(0)),
            batch = small_int(name, "B", B), inter = truth(a[10]) ? 1 : 0;
  const float *c = static_cast<const float*>(ptr(cos)), *s = static_cast<const float*>(ptr(sin));
  const int32_t *tab = static_cast<const int32_t*>(ptr(tables)), *pos = static_cast<const int32_t*>(ptr(positions)),
                *lens = static_cast<const int32_t*>(ptr(cu));
  int32_t* word = static_cast<int32_t*>(mut(err));
  if (int4)
    check(f_rope_append_int4(ptr(q), qs.first, qs.second, ptr(k), ks.first, ks.second, ptr(v), vs.first, vs.second, mut(out),
                             c, s, mut(pool), tab, pos, lens, N, batch, Hq, Hkv, D, rot, inter, max_pos, bs, max_blocks,
                             blocks, code, word, stream()),
          name);
  else
    check(f_rope_append(ptr(q), qs.first, qs.second, ptr(k), ks.first, ks.second, ptr(v), vs.first, vs.second, mut(out), c,
                        s, mut(pool), mut(v_pool), tab, pos, lens, N, batch, Hq, Hkv, D, rot, inter, max_pos, bs,
                        max_blocks, blocks, code, word, stream()),
          name);
  return out;
}

// (pool, block_tables, cu_seqlens, total, head_dim, dtype, starts, k_out, v_out, error_word)
std::pair<at::Tensor, at::Tensor> gather(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 10);
  const at::Tensor &pool = tensor(name, "pool", a[0]), &tables = tensor(name, "block_tables", a[1]),
                   &cu = tensor(name, "cu_seqlens", a[2]), &starts = tensor(name, "starts", a[6], true),
                   &k_given = tensor(name, "k_out", a[7], true), &v_given = tensor(name, "v_out", a[8], true),
                   &err = tensor(name, "error_word", a[9], true);
  current_device(name, {&pool, &tables, &cu, &starts, &k_given, &v_given, &err});
  const int64_t total = PyLong_AsLongLong(a[3]), head_dim = PyLong_AsLongLong(a[4]);
  if (PyErr_Occurred() || !THPDtype_Check(a[5])) {
    PyErr_Clear();
    refuse(name, "total and head_dim must be integers and dtype a torch.dtype");
  }
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  const int code = dtype_code(name, type), N = small_int(name, "total", total), D = small_int(name, "head_dim", head_dim);
  const int Hkv = pool.dim() == 3 ? small_int(name, "Hkv", pool.size(1)) : -1;
  const int bs = int4_block_size(name, pool, Hkv, D);
  const int64_t B = cu.dim() == 1 ? cu.size(0) - 1 : -1;
  int32_vector(name, "cu_seqlens", cu, B + 1);
  if (starts.defined()) int32_vector(name, "starts", starts, B);
  const int max_blocks = table_columns(name, tables, B);
  error_word(name, err);
  const std::array<int64_t, 3> shape{N, Hkv, D};
  auto output = [&](const at::Tensor& given) {
    if (!given.defined()) return at::empty(shape, pool.options().dtype(type));
    if (given.sizes() != at::IntArrayRef(shape) || given.scalar_type() != type || !given.is_contiguous())
      refuse(name, "outputs must be contiguous (", N, ", ", Hkv, ", ", D, ") tensors of ", c10::toString(type));
    return given;
  };
  at::Tensor k, v;
  if (!k_given.defined() && !v_given.defined()) {  // one allocation for both
    const at::Tensor both = at::empty({2, N, Hkv, D}, pool.options().dtype(type));
    k = both.select(0, 0);
    v = both.select(0, 1);
  } else {
    k = output(k_given);
    v = output(v_given);
    if (overlap(k, v)) refuse(name, "k_out and v_out overlap");
  }
  check(f_gather(ptr(pool), static_cast<const int32_t*>(ptr(tables)), static_cast<const int32_t*>(ptr(cu)),
                 static_cast<const int32_t*>(ptr(starts)), mut(k), mut(v), N, small_int(name, "B", B), Hkv, D, bs, max_blocks,
                 small_int(name, "num_blocks", pool.size(0)), code, static_cast<int32_t*>(mut(err)), stream()),
        name);
  return {k, v};
}

// Workspaces of calls that bring none: one per device, stream and graph
// capture, for all operators, made anew when a call needs more arrival counters or partial results than it has room for.
// Counters lie at its start and are left at zero by every call, partial results at its end, so one
// workspace serves all geometries.  One that is made during a capture lies in the graph's memory and is
// zeroed by a node of that graph: it serves that capture's calls and no others, and is let go (back to
// the graph's memory) once kCaptures later ones have come.
constexpr size_t kCaptures = 8, kHeader = 256;
struct Workspace {
  int dev;
  void* stream;
  uint64_t capture;  // 0: outside captures
  size_t counters, partials;  // bytes
  at::Tensor bytes;
};
at::Tensor kept_workspace(const char* name, int dev, void* stream, size_t counters, size_t need, const at::Tensor& like) {
  static auto* kept = new std::vector<Workspace>();  // in the order of their captures
  if (need == 0) refuse(name, "unsupported geometry");
  size_t partials = need - kHeader - counters;
  const uint64_t capture = f_capture_id(stream);
  for (auto e = kept->begin(); e != kept->end(); ++e)
    if (e->dev == dev && e->stream == stream && e->capture == capture) {
      if (e->counters >= counters && e->partials >= partials) return e->bytes;
      counters = std::max(counters, e->counters);
      partials = std::max(partials, e->partials);
      kept->erase(e);
      break;
    }
  if (capture) {
    size_t others = 0;
    uint64_t last = capture;
    for (auto e = kept->rbegin(); e != kept->rend(); ++e)
      if (e->capture && e->capture != capture && e->capture != last) last = e->capture, ++others;
    if (others >= kCaptures) {
      const auto oldest = std::find_if(kept->begin(), kept->end(), [&](const Workspace& e) { return e.capture; })->capture;
      kept->erase(std::remove_if(kept->begin(), kept->end(), [&](const Workspace& e) { return e.capture == oldest; }),
                  kept->end());
    }
  }
  at::Tensor ws = at::empty({(int64_t)(kHeader + counters + partials)}, like.options().dtype(at::kByte));
  ws.narrow(0, 0, (int64_t)(kHeader + counters)).zero_();
  kept->push_back({dev, stream, capture, counters, partials, ws});
  return ws;
}

// (q, pool, block_tables, context_lens, scale, out, workspace, error_word)
at::Tensor decode(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 8);
  const at::Tensor &q = tensor(name, "q", a[0]), &pool = tensor(name, "pool", a[1]), &tables = tensor(name, "block_tables", a[2]),
                   &lens = tensor(name, "context_lens", a[3]), &given = tensor(name, "out", a[5], true),
                   &ws_given = tensor(name, "workspace", a[6], true), &err = tensor(name, "error_word", a[7], true);
  const int dev = current_device(name, {&q, &pool, &tables, &lens, &given, &ws_given, &err});
  if (q.dim() != 3 || !q.is_contiguous()) refuse(name, "q must be a contiguous [B, Hq, D] tensor");
  const int B = small_int(name, "B", q.size(0)), Hq = small_int(name, "Hq", q.size(1)), D = small_int(name, "D", q.size(2));
  const int Hkv = pool.dim() == 3 ? small_int(name, "Hkv", pool.size(1)) : -1;
  const int bs = int4_block_size(name, pool, Hkv, D);
  if (Hkv <= 0 || Hq % Hkv) refuse(name, Hq, " query heads do not divide over ", Hkv, " key/value heads");
  const int max_blocks = table_columns(name, tables, B);
  int32_vector(name, "context_lens", lens, B);
  if (given.defined() && (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !given.is_contiguous()))
    refuse(name, "out must be a contiguous ", shape_of(q), " tensor of q's dtype");
  if (given.defined() && partly_over(q, given)) refuse(name, "out must be apart from q, or q itself");
  error_word(name, err);
  const int code = dtype_code(name, q.scalar_type());
  const double scale = PyFloat_AsDouble(a[4]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, "scale must be a number");
  }
  at::Tensor out = given.defined() ? given : at::empty(q.sizes(), q.options());
  if (B == 0) return out;
  void* st = stream();
  if (ws_given.defined() && (ws_given.scalar_type() != at::kByte || !ws_given.is_contiguous()))
    refuse(name, "workspace must be a contiguous uint8 tensor");
  const size_t counters = ((size_t)B * Hq * 4 + kHeader - 1) / kHeader * kHeader;  // the library's layout
  const at::Tensor ws = ws_given.defined()
                            ? ws_given
                            : kept_workspace(name, dev, st, counters, f_decode_size(B, Hq, Hkv, D, bs, max_blocks, code, dev), q);
  check(f_decode(ptr(q), ptr(pool), static_cast<const int32_t*>(ptr(tables)), static_cast<const int32_t*>(ptr(lens)), mut(out),
                 B, Hq, Hkv, D, bs, max_blocks, small_int(name, "num_blocks", pool.size(0)), (float)scale, code, mut(ws),
                 (size_t)ws.numel(), static_cast<int32_t*>(mut(err)), st),
        name);
  return out;
}

// (q, k, v, cu_seqlens_q, cu_seqlens_k, causal, scale, out, error_word)
at::Tensor prompt(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 9);
  const at::Tensor &q = tensor(name, "q", a[0]), &k = tensor(name, "k", a[1]), &v = tensor(name, "v", a[2]),
                   &cu_q = tensor(name, "cu_seqlens_q", a[3]), &cu_given = tensor(name, "cu_seqlens_k", a[4], true),
                   &given = tensor(name, "out", a[7], true), &err = tensor(name, "error_word", a[8], true);
  const at::Tensor& cu_k = cu_given.defined() ? cu_given : cu_q;
  current_device(name, {&q, &k, &v, &cu_q, &cu_k, &given, &err});
  if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || q.size(2) != k.size(2))
    refuse(name, "q [Nq, Hq, D] and k, v [Nk, Hkv, D] expected");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse(name, "q, k and v must share a dtype");
  const int Nq = small_int(name, "Nq", q.size(0)), Hq = small_int(name, "Hq", q.size(1)), D = small_int(name, "D", q.size(2)),
            Nk = small_int(name, "Nk", k.size(0)), Hkv = small_int(name, "Hkv", k.size(1));
  if (Hkv == 0 || Hq % Hkv) refuse(name, Hq, " query heads do not divide over ", Hkv, " key/value heads");
  const int64_t B = cu_q.dim() == 1 ? cu_q.size(0) - 1 : -1;
  int32_vector(name, "cu_seqlens_q", cu_q, B + 1);
  int32_vector(name, "cu_seqlens_k", cu_k, B + 1);
  if (given.defined() && (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !given.is_contiguous()))
    refuse(name, "out must be a contiguous ", shape_of(q), " tensor of q's dtype");
  // in place of q itself a CTA writes only rows that no other reads
  if (given.defined() && (overlap(k, given) || overlap(v, given) || partly_over(q, given)))
    refuse(name, "out must be apart from k and v, and from q unless it is q itself");
  error_word(name, err);
  const double scale = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, "scale must be a number");
  }
  const int code = dtype_code(name, q.scalar_type());
  const auto qs = token_strides(name, "q", q), ks = token_strides(name, "k", k), vs = token_strides(name, "v", v);
  at::Tensor out = given.defined() ? given : at::empty(q.sizes(), q.options());
  check(f_prompt(ptr(q), qs.first, qs.second, ptr(k), ks.first, ks.second, ptr(v), vs.first, vs.second, mut(out),
                 static_cast<const int32_t*>(ptr(cu_q)), static_cast<const int32_t*>(ptr(cu_k)), Nq, Nk,
                 small_int(name, "B", B), Hq, Hkv, D, truth(a[5]) ? 1 : 0, (float)scale, code,
                 static_cast<int32_t*>(mut(err)), stream()),
        name);
  return out;
}

double number(const char* name, const char* what, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, what, " must be a number");
  }
  return v;
}

void workspace_bytes(const char* name, const at::Tensor& ws) {
  if (ws.defined() && (ws.scalar_type() != at::kByte || !ws.is_contiguous()))
    refuse(name, "workspace must be a contiguous uint8 tensor");
}

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(ptr(t)); }

// (q, k_pool, v_pool, prefix_tables, prefix_lens, cu_groups, block_tables, context_lens, scale, out, workspace, error_word)
at::Tensor prefix(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 12);
  const at::Tensor &q = tensor(name, "q", a[0]), &k = tensor(name, "k_pool", a[1]), &v = tensor(name, "v_pool", a[2]),
                   &ptab = tensor(name, "prefix_tables", a[3], true), &plens = tensor(name, "prefix_lens", a[4], true),
                   &cu = tensor(name, "cu_groups", a[5], true), &tables = tensor(name, "block_tables", a[6]),
                   &lens = tensor(name, "context_lens", a[7]), &given = tensor(name, "out", a[9], true),
                   &ws_given = tensor(name, "workspace", a[10], true), &err = tensor(name, "error_word", a[11], true);
  const int dev = current_device(name, {&q, &k, &v, &ptab, &plens, &cu, &tables, &lens, &given, &ws_given, &err});
  if (q.dim() != 3 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(3) != q.size(2))
    refuse(name, "q [B, Hq, D] and pools [num_blocks, block_size, Hkv, D] expected");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse(name, "q and the pools must share a dtype");
  if (!k.is_contiguous() || !v.is_contiguous()) refuse(name, "pools must be contiguous");
  const int B = small_int(name, "B", q.size(0)), Hq = small_int(name, "Hq", q.size(1)), D = small_int(name, "D", q.size(2)),
            bs = small_int(name, "block_size", k.size(1)), Hkv = small_int(name, "Hkv", k.size(2)),
            blocks = small_int(name, "num_blocks", k.size(0));
  if (Hkv == 0 || Hq % Hkv) refuse(name, Hq, " query heads do not divide over ", Hkv, " key/value heads");
  const int max_blocks = table_columns(name, tables, B);
  int32_vector(name, "context_lens", lens, B);
  if (ptab.defined() != plens.defined() || ptab.defined() != cu.defined())
    refuse(name, "prefix_tables, prefix_lens and cu_groups come together");
  int G = 0, max_prefix = 0;
  if (ptab.defined()) {
    if (ptab.dim() != 2 || ptab.scalar_type() != at::kInt || !ptab.is_contiguous())
      refuse(name, "prefix_tables must be contiguous int32 [G, max_prefix_blocks]");
    G = small_int(name, "G", ptab.size(0));
    max_prefix = small_int(name, "max_prefix_blocks", ptab.size(1));
    int32_vector(name, "prefix_lens", plens, G);
    int32_vector(name, "cu_groups", cu, (int64_t)G + 1);
  }
  if (given.defined() && (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !given.is_contiguous()))
    refuse(name, "out must be a contiguous ", shape_of(q), " tensor of q's dtype");
  if (given.defined() && (overlap(k, given) || overlap(v, given) || partly_over(q, given)))
    refuse(name, "out must be apart from the pools, and from q unless it is q itself");
  error_word(name, err);
  workspace_bytes(name, ws_given);
  const int code = dtype_code(name, q.scalar_type());
  const double scale = number(name, "scale", a[8]);
  const auto qs = token_strides(name, "q", q);
  at::Tensor out = given.defined() ? given : at::empty(q.sizes(), q.options());
  if (B == 0) return out;
  void* st = stream();
  at::Tensor ws = ws_given;
  if (!ws.defined()) {
    const size_t need = f_prefix_size(B, G, Hq, Hkv, D, bs, max_prefix, max_blocks, dev);
    const size_t counters = ((size_t)B * Hq * 4 + kHeader - 1) / kHeader * kHeader;  // as much as the library's, or more
    ws = kept_workspace(name, dev, st, counters, need ? need + counters : 0, q);
  }
  check(f_prefix(ptr(q), qs.first, qs.second, ptr(k), ptr(v), ints(ptab), ints(plens), ints(cu), ints(tables), ints(lens),
                 mut(out), B, G, Hq, Hkv, D, bs, max_prefix, max_blocks, blocks, (float)scale, code, mut(ws),
                 (size_t)ws.numel(), static_cast<int32_t*>(mut(err)), st),
        name);
  return out;
}

// (q, k, v, valid_lens, cu_seqlens, slot_ids, scale, out, workspace, error_word)
at::Tensor cross(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 10);
  const at::Tensor &q = tensor(name, "q", a[0]), &k = tensor(name, "k", a[1]), &v = tensor(name, "v", a[2]),
                   &lens = tensor(name, "valid_lens", a[3]), &cu = tensor(name, "cu_seqlens", a[4], true),
                   &slots = tensor(name, "slot_ids", a[5], true), &given = tensor(name, "out", a[7], true),
                   &ws_given = tensor(name, "workspace", a[8], true), &err = tensor(name, "error_word", a[9], true);
  const int dev = current_device(name, {&q, &k, &v, &lens, &cu, &slots, &given, &ws_given, &err});
  if (q.dim() != 3 || k.dim() != 4 || v.sizes() != k.sizes() || k.size(3) != q.size(2))
    refuse(name, "q [N, Hq, D] and k, v [S, Hkv, T, D] expected");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse(name, "q, k and v must share a dtype");
  const int N = small_int(name, "N", q.size(0)), Hq = small_int(name, "Hq", q.size(1)), D = small_int(name, "D", q.size(2)),
            S = small_int(name, "S", k.size(0)), Hkv = small_int(name, "Hkv", k.size(1)), T = small_int(name, "T", k.size(2));
  if (Hkv == 0 || Hq % Hkv) refuse(name, Hq, " query heads do not divide over ", Hkv, " key/value heads");
  if (lens.dim() != 1) refuse(name, "valid_lens must be a contiguous int32 [B] tensor");
  const int B = small_int(name, "B", lens.size(0));
  int32_vector(name, "valid_lens", lens, B);
  if (cu.defined()) int32_vector(name, "cu_seqlens", cu, (int64_t)B + 1);
  else if (N != B) refuse(name, "without cu_seqlens one query per request is expected (", N, " queries, ", B, " requests)");
  if (slots.defined()) int32_vector(name, "slot_ids", slots, B);
  else if (B > S) refuse(name, "more requests than slots and no slot_ids");
  // strides of dimensions of one entry, which nothing steps over, are taken as dense
  int64_t st_[2][3];
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& x = i ? v : k;
    if (x.stride(3) != 1 && D > 1) refuse(name, "k and v need a contiguous last dimension");
    st_[i][2] = T == 1 ? D : x.stride(2);
    st_[i][1] = Hkv == 1 ? st_[i][2] * T : x.stride(1);
    st_[i][0] = S == 1 ? st_[i][1] * Hkv : x.stride(0);
  }
  for (int i = 0; i < 3; ++i)
    if (st_[0][i] != st_[1][i]) refuse(name, "k and v need identical strides");
  if (given.defined() && (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !given.is_contiguous()))
    refuse(name, "out must be a contiguous ", shape_of(q), " tensor of q's dtype");
  if (given.defined() && (overlap(k, given) || overlap(v, given) || partly_over(q, given)))
    refuse(name, "out must be apart from k and v, and from q unless it is q itself");
  error_word(name, err);
  workspace_bytes(name, ws_given);
  const int code = dtype_code(name, q.scalar_type());
  const double scale = number(name, "scale", a[6]);
  const auto qs = token_strides(name, "q", q);
  at::Tensor out = given.defined() ? given : at::empty(q.sizes(), q.options());
  if (N == 0 || B == 0) return out;
  void* st = stream();
  at::Tensor ws = ws_given;
  if (!ws.defined()) ws = kept_workspace(name, dev, st, 0, f_cross_size(N, Hq, Hkv, D, dev), q);
  check(f_cross(ptr(q), qs.first, qs.second, ptr(k), ptr(v), st_[0][0], st_[0][1], st_[0][2], ints(lens), ints(cu), ints(slots),
                mut(out), N, B, S, T, Hq, Hkv, D, (float)scale, code, mut(ws), (size_t)ws.numel(),
                static_cast<int32_t*>(mut(err)), st),
        name);
  return out;
}

// A setting of sample_rows: a number for all rows, or a tensor with one for each.
struct Setting {
  const void* rows = nullptr;
  double all = 0.0;
};
Setting setting(const char* name, const char* what, PyObject* o, int64_t rows, at::ScalarType type) {
  Setting s;
  if (!THPVariable_Check(o)) {
    s.all = number(name, what, o);
    return s;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != rows || !t.is_contiguous())
    refuse(name, what, " must be a number or a contiguous ", c10::toString(type), " [", rows, "] tensor");
  s.rows = ptr(t);
  return s;
}

// (x, uniforms, temperature, top_k, top_p, min_p, cols, skip, out, logprobs)
at::Tensor sample(const char* name, PyObject* const* a, Py_ssize_t n_args) {
  count(name, n_args, 10);
  const at::Tensor &x = tensor(name, "x", a[0]), &u = tensor(name, "uniforms", a[1]), &skip = tensor(name, "skip", a[7], true),
                   &given = tensor(name, "out", a[8], true), &logs = tensor(name, "logprobs", a[9], true);
  std::vector<const at::Tensor*> all{&x, &u, &skip, &given, &logs};
  for (int i = 2; i < 6; ++i)
    if (THPVariable_Check(a[i])) all.push_back(&THPVariable_Unpack(a[i]));
  for (const at::Tensor* t : all) current_device(name, {t});
  if (x.dim() != 2 || (x.stride(1) != 1 && x.size(1) > 1)) refuse(name, "x must be [rows, ld] with unit column stride");
  const int rows = small_int(name, "rows", x.size(0));
  int64_t cols = x.size(1);
  if (a[6] != Py_None) {
    cols = PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      refuse(name, "cols must be an integer");
    }
  }
  if (cols <= 0 || cols > x.size(1)) refuse(name, "cols ", cols, " outside [1, ", x.size(1), "]");
  if (u.scalar_type() != at::kFloat || u.dim() != 1 || u.size(0) != rows || !u.is_contiguous())
    refuse(name, "uniforms must be a contiguous float32 [", rows, "] tensor");
  if (skip.defined() && (skip.scalar_type() != at::kBool || skip.numel() < cols || !skip.is_contiguous()))
    refuse(name, "skip must be a contiguous bool mask of at least cols entries");
  const Setting t = setting(name, "temperature", a[2], rows, at::kFloat), k = setting(name, "top_k", a[3], rows, at::kInt),
                tp = setting(name, "top_p", a[4], rows, at::kFloat), mp = setting(name, "min_p", a[5], rows, at::kFloat);
  if (!(k.all >= INT32_MIN && k.all <= INT32_MAX) || k.all != (double)(int)k.all) refuse(name, "top_k must be a whole number");
  if (given.defined() && (given.scalar_type() != at::kLong || given.dim() != 1 || given.size(0) != rows || !given.is_contiguous()))
    refuse(name, "out must be a contiguous int64 [", rows, "] tensor");
  if (logs.defined() && (logs.scalar_type() != at::kFloat || logs.dim() != 1 || logs.size(0) != rows || !logs.is_contiguous()))
    refuse(name, "logprobs must be a contiguous float32 [", rows, "] tensor");
  const int code = dtype_code(name, x.scalar_type());
  const at::Tensor out = given.defined() ? given : at::empty({rows}, x.options().dtype(at::kLong));
  for (size_t i = 0; i < all.size(); ++i)  // (3: out itself, 4: logprobs; one tensor may stand in two places)
    if (all[i]->defined() && ((i != 3 && overlap(out, *all[i])) || (i != 4 && logs.defined() && overlap(logs, *all[i]))))
      refuse(name, "out and logprobs must be apart from all else");
  const int64_t ld = rows > 1 ? x.stride(0) : x.size(1);
  if (ld < cols) refuse(name, "rows of x overlap");
  check(f_sample(ptr(x), rows, (int)cols, ld, static_cast<const uint8_t*>(ptr(skip)), static_cast<const float*>(ptr(u)),
                 static_cast<const float*>(t.rows), (float)t.all, static_cast<const int32_t*>(k.rows), (int)k.all,
                 static_cast<const float*>(tp.rows), (float)tp.all, static_cast<const float*>(mp.rows), (float)mp.all,
                 static_cast<int64_t*>(mut(out)), static_cast<float*>(mut(logs)), code, stream()),
        name);
  return out;
}

// Runs `body` with every C++ exception turned into a Python RuntimeError.
template <typename F>
PyObject* guarded(const F& body) {
  try {
    return body();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

PyObject* py_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(rope_append("rope_kv_append", false, a, n)); });
}
PyObject* py_rope_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(rope_append("rope_kv_append_int4", true, a, n)); });
}
PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const auto kv = gather("kv_gather_int4", a, n);
    PyObject *k = wrap(kv.first), *v = wrap(kv.second);
    PyObject* both = k && v ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return both;
  });
}
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(decode("paged_decode_attn_int4", a, n)); });
}
PyObject* py_prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(prompt("prompt_attn", a, n)); });
}
PyObject* py_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(prefix("shared_prefix_attn", a, n)); });
}
PyObject* py_sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(sample("sample_rows", a, n)); });
}
PyObject* py_cross(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] { return wrap(cross("cross_attn_packed", a, n)); });
}

// setup({name: address}) of the C ABI's functions
PyObject* py_setup(PyObject*, PyObject* d) {
  auto get = [&](const char* name, auto& f) {
    PyObject* o = PyDict_Check(d) ? PyDict_GetItemString(d, name) : nullptr;
    void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
    if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "setup: no address of %s", name);
    f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
    return p != nullptr;
  };
  if (get("spd_rope_kv_append", f_rope_append) && get("spd_rope_kv_append_int4", f_rope_append_int4) &&
      get("spd_kv_gather_int4", f_gather) && get("spd_paged_decode_attn_int4_err", f_decode) &&
      get("spd_paged_decode_attn_int4_workspace_size", f_decode_size) && get("spd_prompt_attn", f_prompt) &&
      get("spd_kv_int4_page_bytes", f_page_bytes) && get("spd_get_last_error", f_last_error) &&
      get("spd_stream_capture_id", f_capture_id) && get("spd_shared_prefix_attn", f_prefix) &&
      get("spd_shared_prefix_attn_workspace_size", f_prefix_size) && get("spd_cross_attn_packed", f_cross) &&
      get("spd_sample_rows", f_sample) &&
      get("spd_cross_attn_packed_workspace_size", f_cross_size))
    Py_RETURN_NONE;
  return nullptr;
}

PyMethodDef methods[] = {
    {"setup", py_setup, METH_O, "Takes the addresses of the C ABI's functions."},
    {"rope_kv_append", reinterpret_cast<PyCFunction>(py_rope), METH_FASTCALL, nullptr},
    {"rope_kv_append_int4", reinterpret_cast<PyCFunction>(py_rope_int4), METH_FASTCALL, nullptr},
    {"kv_gather_int4", reinterpret_cast<PyCFunction>(py_gather), METH_FASTCALL, nullptr},
    {"paged_decode_attention_int4", reinterpret_cast<PyCFunction>(py_decode), METH_FASTCALL, nullptr},
    {"prompt_attention", reinterpret_cast<PyCFunction>(py_prompt), METH_FASTCALL, nullptr},
    {"shared_prefix_decode_attention", reinterpret_cast<PyCFunction>(py_prefix), METH_FASTCALL, nullptr},
    {"sample_rows", reinterpret_cast<PyCFunction>(py_sample), METH_FASTCALL, nullptr},
    {"cross_attention_packed", reinterpret_cast<PyCFunction>(py_cross), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "spd_torch", "torch tensors to the C ABI of libspd_b200.so", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_spd_torch() { return PyModule_Create(&module); }
