// Python binding of the 4-bit cache's operators: checks the tensors and calls
// the C ABI (include/flexkv_b200.h).  A CPython module on torch's C++ tensors
// and not ctypes, because these run once per layer and token: reading the
// tensors' shapes in Python and converting up to 29 arguments took 15 to 20 us
// a call, several times the smallest kernels; here it takes 2.5 us, nearly all of
// them the launch, and about 1 us for each tensor it allocates.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/flexkv_b200.h"
#include "fp4_overlap.h"

namespace {

using at::Tensor;

// The library's entry points, of the copy that flexkv_b200._lib has loaded.
struct {
  decltype(&::fkv_last_error) last_error;
  decltype(&::fkv_fp4_write) write;
  decltype(&::fkv_fp4_read) read;
  decltype(&::fkv_fp4_pack_blocks) pack_blocks;
  decltype(&::fkv_fp4_unpack_blocks) unpack_blocks;
  decltype(&::fkv_fp4_pack_blocks_listed) pack_blocks_listed;
  decltype(&::fkv_fp4_unpack_blocks_listed) unpack_blocks_listed;
  decltype(&::fkv_fp4_attention_workspace) attention_workspace;
  decltype(&::fkv_fp4_attention) attention;
} lib;

struct StatusError {
  int code;
  const char *where;
};

template <typename... T>
[[noreturn]] void refuse(const T &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw std::runtime_error(s.str());
}

void check(int rc, const char *where) {
  if (rc != FKV_OK) throw StatusError{rc, where};
}

const Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
const Tensor *optional_tensor(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

struct Geometry {
  int64_t blocks, kv_stride, block_stride;
  int kv, tpb, heads, dim;
};

Geometry geometry(const Tensor &t, const char *name) {
  if (t.scalar_type() != at::kByte || t.dim() != 5)
    refuse(name, " must be a uint8 tensor [kv, blocks, heads, tokens_per_block / 16, 9 * head_size]");
  const auto n = t.sizes(), s = t.strides();
  if ((n[0] != 1 && n[0] != 2) || n[2] <= 0 || n[3] <= 0 || n[4] <= 0 || n[4] % 144 || n[2] > 65536 || n[3] > 1 << 20 ||
      n[4] > 9 * 65536)
    refuse(name,
           " must be [kv, blocks, heads, tokens_per_block / 16, 9 * head_size] with kv 1 or 2 and head_size a multiple "
           "of 16, got ", n);
  if (s[4] != 1 || (n[3] > 1 && s[3] != n[4]) || (n[2] > 1 && s[2] != n[3] * n[4]))
    refuse(name, ": a block must be contiguous");
  if (!t.is_cuda()) refuse(name, " must be a CUDA tensor");
  // an axis of one entry is never stepped along: its stride says nothing
  return {n[1], n[0] > 1 ? s[0] : 0, n[1] > 1 ? s[1] : 0, (int)n[0], (int)n[3] * 16, (int)n[2], (int)(n[4] / 9)};
}

int64_t block_bytes(const Geometry &g) { return (int64_t)g.heads * g.tpb * g.dim / 16 * 9; }

int dtype_code(at::ScalarType t, const char *name) {
  if (t == at::kBFloat16) return FKV_DTYPE_BF16;
  if (t == at::kHalf) return FKV_DTYPE_FP16;
  refuse(name, " must be bfloat16 or half, got ", t);
}

void on_device(const Tensor &t, const char *name, const at::Device &dev) {
  if (t.device() != dev) refuse(name, " must be on ", dev, ", got ", t.device());
}

void indices(const Tensor &t, const char *name, at::ScalarType type, const at::Device &dev, int dim = 1) {
  if (t.scalar_type() != type || t.dim() != dim) refuse(name, " must be a ", dim, "-D ", type, " tensor");
  on_device(t, name, dev);
}

struct Rows {
  int64_t token = 0, head = 0;  // strides in bytes
};

Rows rows(const Tensor &t, const char *name, int64_t tokens, int64_t heads, int64_t dim, at::ScalarType type,
          const at::Device &dev) {
  if (t.scalar_type() != type || t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != dim)
    refuse(name, " must be a ", type, " tensor of shape [", tokens, ", ", heads, ", ", dim, "]");
  on_device(t, name, dev);
  if (t.stride(2) != 1) refuse(name, ": the channels of a head must be contiguous");
  return {tokens > 1 ? 2 * t.stride(0) : 0, heads > 1 ? 2 * t.stride(1) : 0};
}

// What a call writes must not overlap itself.
void rows_apart(const Tensor &t, const char *name) {
  const int64_t token = t.stride(0), head = t.stride(1), D = t.size(2), n = t.size(0), heads = t.size(1);
  if (n <= 1 && heads <= 1) return;
  const bool heads_inside = heads <= 1 || (head >= D && (n <= 1 || token >= (heads - 1) * head + D));
  const bool tokens_inside = n <= 1 || (token >= D && (heads <= 1 || head >= (n - 1) * token + D));
  if (!heads_inside && !tokens_inside) refuse(name, ": rows overlap");
}
// The rows of t as a set, for two outputs or an input and an output.
fkv::RowSet row_set(const Tensor &t, const Rows &r) {
  return {(uintptr_t)t.data_ptr(), t.size(0), t.size(1), r.token, r.head, 2 * t.size(2)};
}
void blocks_apart(const Tensor &t, int64_t block, const char *name) {
  const int64_t kv = t.stride(0), blk = t.stride(1), n = t.size(1), sides = t.size(0);
  if (n <= 1 && sides <= 1) return;
  const bool sides_inside = sides <= 1 || (kv >= block && (n <= 1 || blk >= (sides - 1) * kv + block));
  const bool blocks_inside = n <= 1 || (blk >= block && (sides <= 1 || kv >= (n - 1) * blk + block));
  if (!sides_inside && !blocks_inside) refuse(name, ": blocks overlap");
}

// Nothing here is differentiable: what records a gradient, or carries a tangent, is refused.
void no_grad(std::initializer_list<const Tensor *> ts) {
  const bool backward = c10::GradMode::is_enabled();
  const bool forward = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;  // else there are no tangents
  for (const Tensor *t : ts) {
    if (!t) continue;
    if (backward && t->requires_grad()) refuse("the 4-bit cache has no gradient: call under torch.no_grad()");
    if (forward && t->_fw_grad(0).defined()) refuse("the 4-bit cache has no gradient: an input has a tangent");
  }
}

// After a call that writes t: a backward pass that kept its old content must not run.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void *stream_of(const at::Device &dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void *data(const Tensor *t) { return t ? t->data_ptr() : nullptr; }

// Runs a call and turns what it throws into a Python exception.
template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const StatusError &e) {
    PyObject *mod = PyImport_ImportModule("flexkv_b200._lib");
    PyObject *type = mod ? PyObject_GetAttrString(mod, "FlexKVError") : nullptr;
    PyObject *error = type ? PyObject_CallFunction(type, "iss", e.code, e.where, lib.last_error()) : nullptr;
    if (error) PyErr_SetObject(type, error);
    Py_XDECREF(error);
    Py_XDECREF(type);
    Py_XDECREF(mod);
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

bool count(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
  return false;
}

// write(layer, k, v, slot_mapping)
PyObject *write(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count(n, 4)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Tensor &layer = tensor(args[0], "layer"), &k = tensor(args[1], "k"), &slots = tensor(args[3], "slot_mapping");
    const Tensor *v = optional_tensor(args[2], "v");
    const Geometry g = geometry(layer, "layer");
    no_grad({&k, v});
    const at::Device dev = layer.device();
    indices(slots, "slot_mapping", at::kLong, dev);
    const int64_t tokens = slots.size(0);
    if ((v == nullptr) != (g.kv == 1))
      refuse("v must be given for a layer of keys and values, and None for a latent layer");
    const int dt = dtype_code(k.scalar_type(), "k");
    const Rows rk = rows(k, "k", tokens, g.heads, g.dim, k.scalar_type(), dev);
    const Rows rv = v ? rows(*v, "v", tokens, g.heads, g.dim, k.scalar_type(), dev) : Rows{};
    blocks_apart(layer, block_bytes(g), "layer");
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor ids = slots.contiguous();
    check(lib.write(layer.data_ptr(), g.kv, g.blocks, g.tpb, g.heads, g.dim, g.kv_stride, g.block_stride, k.data_ptr(),
                        data(v), rk.token, rk.head, rv.token, rv.head, dt, ids.data_ptr<int64_t>(), tokens, stream_of(dev)),
          "fp4_write");
    written(layer);
    Py_RETURN_NONE;
  });
}

// read(layer, slot_mapping, dtype, k or None, v or None) -> (k, v)
PyObject *read(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count(n, 5)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Tensor &layer = tensor(args[0], "layer"), &slots = tensor(args[1], "slot_mapping");
    const Geometry g = geometry(layer, "layer");
    const at::Device dev = layer.device();
    indices(slots, "slot_mapping", at::kLong, dev);
    const int64_t tokens = slots.size(0);
    if (!THPDtype_Check(args[2])) refuse("dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype *>(args[2])->scalar_type;
    const int dt = dtype_code(type, "dtype");
    const c10::cuda::CUDAGuard guard(dev);
    Tensor k, v;
    if (args[3] == Py_None) {
      const auto options = layer.options().dtype(type);
      k = at::empty({tokens, g.heads, g.dim}, options);
      if (g.kv == 2) v = at::empty({tokens, g.heads, g.dim}, options);
    } else {
      k = tensor(args[3], "k");
      if (const Tensor *t = optional_tensor(args[4], "v")) v = *t;
      if (v.defined() != (g.kv == 2))
        refuse("out must hold v for a layer of keys and values, and None for a latent layer");
      no_grad({&k, v.defined() ? &v : nullptr});
    }
    const Rows rk = rows(k, "k", tokens, g.heads, g.dim, type, dev);
    const Rows rv = v.defined() ? rows(v, "v", tokens, g.heads, g.dim, type, dev) : Rows{};
    if (args[3] != Py_None) {
      rows_apart(k, "k");
      if (v.defined()) {
        rows_apart(v, "v");
        if (fkv::rows_share_memory(row_set(k, rk), row_set(v, rv))) refuse("k and v overlap");
      }
    }
    const Tensor ids = slots.contiguous();
    check(lib.read(layer.data_ptr(), g.kv, g.blocks, g.tpb, g.heads, g.dim, g.kv_stride, g.block_stride, k.data_ptr(),
                       v.defined() ? v.data_ptr() : nullptr, rk.token, rk.head, rv.token, rv.head, dt,
                       ids.data_ptr<int64_t>(), tokens, stream_of(dev)),
          "fp4_read");
    if (args[3] != Py_None) {
      written(k);
      if (v.defined()) written(v);
    }
    PyObject *pk = THPVariable_Wrap(k);
    PyObject *pv = v.defined() ? THPVariable_Wrap(v) : Py_NewRef(Py_None);
    PyObject *out = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return out;
  });
}

// Block ids, contiguous, where they are; host ids are checked.
Tensor block_ids(const Tensor &t, const char *name, int64_t pool, const at::Device &dev, bool distinct) {
  if (t.scalar_type() != at::kLong || t.dim() != 1) refuse(name, " must be a 1-D ", at::kLong, " tensor");
  if (t.is_cuda()) {
    on_device(t, name, dev);
    return t.contiguous();
  }
  if (!t.is_cpu()) refuse(name, " must be on ", dev, " or on the host, got ", t.device());
  const Tensor c = t.contiguous();
  std::vector<int64_t> ids(c.data_ptr<int64_t>(), c.data_ptr<int64_t>() + c.numel());
  for (const int64_t id : ids)
    if (id < 0 || id >= pool) refuse(name, ": block id ", id, " is outside [0, ", pool, ")");
  if (distinct) {
    std::sort(ids.begin(), ids.end());
    if (std::adjacent_find(ids.begin(), ids.end()) != ids.end()) refuse(name, ": a block id appears twice");
  }
  return c;
}

// convert(pack, kv_layers, fp4_layers, kv_block_ids, fp4_block_ids)
PyObject *convert(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count(n, 5)) return nullptr;
  PyObject *kvs = PySequence_Fast(args[1], "kv_layers must be a sequence of tensors");
  PyObject *fps = kvs ? PySequence_Fast(args[2], "fp4_layers must be a sequence of tensors") : nullptr;
  PyObject *out = !fps ? nullptr : guarded([&]() -> PyObject * {
    const bool pack = args[0] == Py_True;
    const Py_ssize_t layers = PySequence_Fast_GET_SIZE(kvs);
    if (layers != PySequence_Fast_GET_SIZE(fps) || layers == 0)
      refuse("kv_layers and fp4_layers must hold the same layers, at least one");
    const Tensor &f0 = tensor(PySequence_Fast_GET_ITEM(fps, 0), "fp4_layers[0]");
    const Tensor &k0 = tensor(PySequence_Fast_GET_ITEM(kvs, 0), "kv_layers[0]");
    const Geometry g = geometry(f0, "fp4_layers[0]");
    const at::Device dev = f0.device();
    if (k0.dim() != 5 || k0.size(0) != g.kv || k0.size(2) != g.tpb || k0.size(3) != g.heads || k0.size(4) != g.dim)
      refuse("a 16-bit layer must be [", g.kv, ", blocks, ", g.tpb, ", ", g.heads, ", ", g.dim, "], got ", k0.sizes());
    const int dt = dtype_code(k0.scalar_type(), "a 16-bit layer");
    if (k0.stride(4) != 1 || (g.heads > 1 && k0.stride(3) != g.dim) || k0.stride(2) != (int64_t)g.heads * g.dim)
      refuse("a block of a 16-bit layer must be contiguous");
    if (pack)
      blocks_apart(f0, block_bytes(g), "fp4_layers");
    else
      blocks_apart(k0, (int64_t)g.tpb * g.heads * g.dim, "kv_layers");
    std::vector<void *> kp(layers), fp(layers);
    std::vector<const Tensor *> targets(layers);
    for (Py_ssize_t i = 0; i < layers; ++i) {
      const Tensor &f = tensor(PySequence_Fast_GET_ITEM(fps, i), "an entry of fp4_layers");
      const Tensor &k = tensor(PySequence_Fast_GET_ITEM(kvs, i), "an entry of kv_layers");
      if (f.scalar_type() != at::kByte || f.sizes() != f0.sizes() || f.strides() != f0.strides() || f.device() != dev)
        refuse("fp4_layers[", i, "] must have the shape, strides and device of fp4_layers[0]");
      if (k.scalar_type() != k0.scalar_type() || k.sizes() != k0.sizes() || k.strides() != k0.strides() || k.device() != dev)
        refuse("kv_layers[", i, "] must have the type, shape and strides of kv_layers[0] and be on ", dev);
      no_grad({&k});
      kp[i] = k.data_ptr(), fp[i] = f.data_ptr(), targets[i] = pack ? &f : &k;
    }
    std::vector<void *> to = pack ? fp : kp;
    // layers that are allocated one after another are in order already
    if (std::adjacent_find(to.begin(), to.end(), std::greater_equal<>()) != to.end()) std::sort(to.begin(), to.end());
    if ((pack ? f0 : k0).numel() && std::adjacent_find(to.begin(), to.end()) != to.end())
      refuse(pack ? "fp4_layers" : "kv_layers", ": a layer to write to appears twice");
    const Tensor &ka = tensor(args[3], "kv_block_ids"), &fa = tensor(args[4], "fp4_block_ids");
    if (ka.numel() != fa.numel()) refuse("kv_block_ids and fp4_block_ids differ in length");
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor kids = block_ids(ka, "kv_block_ids", k0.size(1), dev, !pack);
    const Tensor fids = block_ids(fa, "fp4_block_ids", g.blocks, dev, pack);
    const int host = (kids.is_cuda() ? 0 : FKV_FP4_KV_IDS) | (fids.is_cuda() ? 0 : FKV_FP4_FP4_IDS);
    const int64_t ks = g.kv > 1 ? 2 * k0.stride(0) : 0, kb = k0.size(1) > 1 ? 2 * k0.stride(1) : 0;
    const int64_t n = kids.numel(), *ki = kids.data_ptr<int64_t>(), *fi = fids.data_ptr<int64_t>();
    void *const stream = stream_of(dev);
    const char *const who = pack ? "fp4_pack_blocks" : "fp4_unpack_blocks";
    auto call = [&](auto pack_blocks, auto unpack_blocks, auto... lists) {
      check(pack ? pack_blocks((int)layers, kp.data(), fp.data(), g.kv, g.tpb, g.heads, g.dim, k0.size(1), ks, kb, g.blocks,
                               g.kv_stride, g.block_stride, dt, ki, fi, n, lists..., stream)
                 : unpack_blocks((int)layers, fp.data(), kp.data(), g.kv, g.tpb, g.heads, g.dim, g.blocks, g.kv_stride,
                                 g.block_stride, k0.size(1), ks, kb, dt, fi, ki, n, lists..., stream),
            who);
    };
    if (host)
      call(lib.pack_blocks_listed, lib.unpack_blocks_listed, host);
    else
      call(lib.pack_blocks, lib.unpack_blocks);
    for (const Tensor *t : targets) written(*t);
    Py_RETURN_NONE;
  });
  Py_XDECREF(fps);
  Py_XDECREF(kvs);
  return out;
}

// attention(layer, q, block_tables, seq_lens, cu_seqlens_q, max_q_len, softmax_scale, causal, out, return_lse)
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (!count(nargs, 10)) return nullptr;
  return guarded([&]() -> PyObject * {
    const Tensor &layer = tensor(args[0], "layer"), &q = tensor(args[1], "q"), &tables = tensor(args[2], "block_tables"),
                 &lens = tensor(args[3], "seq_lens");
    const Tensor *cu = optional_tensor(args[4], "cu_seqlens_q"), *given = optional_tensor(args[8], "out");
    const Geometry g = geometry(layer, "layer");
    const at::Device dev = layer.device();
    if (g.kv != 2) refuse("attention reads a layer of keys and values (kv = 2)");
    if (q.dim() != 3) refuse("q must be [tokens, num_q_heads, head_size]");
    const int64_t n = q.size(0), q_heads = q.size(1);
    const int dt = dtype_code(q.scalar_type(), "q");
    const Rows rq = rows(q, "q", n, q_heads, g.dim, q.scalar_type(), dev);
    no_grad({&q, given});
    if (q_heads <= 0 || q_heads % g.heads || q_heads > 1 << 20)
      refuse("num_q_heads (", q_heads, ") must be a multiple of the layer's heads (", g.heads, ")");
    indices(lens, "seq_lens", at::kInt, dev);
    indices(tables, "block_tables", at::kInt, dev, 2);
    const int64_t seqs = lens.size(0);
    if (tables.size(0) != seqs) refuse("block_tables and seq_lens differ in their number of sequences");
    if (seqs > INT32_MAX || n > INT32_MAX || tables.size(1) > INT32_MAX) refuse("2^31 sequences, tokens or pages or more");
    int64_t longest;
    if (cu) {
      indices(*cu, "cu_seqlens_q", at::kInt, dev);
      if (cu->size(0) != seqs + 1) refuse("cu_seqlens_q must have one entry more than seq_lens");
      longest = n;
      if (args[5] != Py_None) {
        const long long m = PyLong_AsLongLong(args[5]);
        if (m == -1 && PyErr_Occurred()) return nullptr;
        if (m < 0) refuse("max_q_len must be non-negative");
        longest = std::min<int64_t>(m, n);
      }
    } else {
      if (seqs ? n % seqs : n) refuse("without cu_seqlens_q every sequence has the same number of rows");
      longest = seqs ? n / seqs : 0;
    }
    double scale = 1 / std::sqrt((double)g.dim);
    if (args[6] != Py_None) {
      scale = PyFloat_AsDouble(args[6]);
      if (scale == -1 && PyErr_Occurred()) return nullptr;
    }
    if (!std::isfinite(scale)) refuse("softmax_scale must be finite");
    const int causal = PyObject_IsTrue(args[7]), want_lse = PyObject_IsTrue(args[9]);
    if (causal < 0 || want_lse < 0) return nullptr;
    const c10::cuda::CUDAGuard guard(dev);
    // without cu_seqlens_q every row belongs to a sequence, and without a sequence nothing is launched
    const bool fill = !given && cu && seqs;
    Tensor out = given           ? *given
                 : cu && !seqs ? at::zeros({n, q_heads, g.dim}, q.options())
                                 : at::empty({n, q_heads, g.dim}, q.options());
    const Rows ro = rows(out, "out", n, q_heads, g.dim, q.scalar_type(), dev);
    if (given) {
      rows_apart(out, "out");
      const fkv::RowSet from = row_set(q, rq), to = row_set(out, ro);
      if (!from.same_place(to) && fkv::rows_share_memory(from, to))
        refuse("out may be q itself, but must not overlap it otherwise");
    }
    Tensor lse;
    if (want_lse)
      lse = cu && !fill ? at::full({n, q_heads}, -INFINITY, q.options().dtype(at::kFloat))
                        : at::empty({n, q_heads}, q.options().dtype(at::kFloat));
    const Tensor t = tables.size(1) > 1 && tables.stride(1) != 1 ? tables.contiguous() : tables;
    const Tensor l = lens.contiguous();
    std::optional<Tensor> c;
    if (cu) c = cu->contiguous();
    const int64_t bytes =
        lib.attention_workspace(n, (int)q_heads, g.heads, g.dim, (int)seqs, (int)longest);
    Tensor workspace;
    if (bytes > 0) workspace = at::empty({bytes}, layer.options());
    check(lib.attention(layer.data_ptr(), g.blocks, g.tpb, g.heads, g.dim, g.kv_stride, g.block_stride, q.data_ptr(),
                            out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, rq.token, rq.head, ro.token, ro.head,
                            dt, n, (int)q_heads, t.data_ptr<int32_t>(), t.stride(0), (int)t.size(1), l.data_ptr<int32_t>(),
                            c ? c->data_ptr<int32_t>() : nullptr, (int)seqs, (int)longest, (float)scale,
                            (causal ? FKV_FP4_CAUSAL : 0) | (fill ? FKV_FP4_FILL_REST : 0),
                            bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(dev)),
          "fp4_attention");
    if (given) written(out);
    PyObject *po = given ? Py_NewRef(args[8]) : THPVariable_Wrap(out);
    if (!want_lse || !po) return po;
    PyObject *pl = THPVariable_Wrap(lse);
    PyObject *both = pl ? PyTuple_Pack(2, po, pl) : nullptr;
    Py_DECREF(po);
    Py_XDECREF(pl);
    return both;
  });
}

// bind(addresses): where the entry points are, in the order of `lib`
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void **at = reinterpret_cast<void **>(&lib);
  if (!count(n, sizeof(lib) / sizeof(void *))) return nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"write", (PyCFunction)(void (*)(void))write, METH_FASTCALL, nullptr},
    {"read", (PyCFunction)(void (*)(void))read, METH_FASTCALL, nullptr},
    {"convert", (PyCFunction)(void (*)(void))convert, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp4", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fp4(void) { return PyModule_Create(&module); }
