// Python calls of the operators around the paged cache (module fgw_amd._kv).
//
// One C++ function per operator: the checks of its tensors, the allocation of outputs and
// workspaces with torch's caching allocator, and the launch through the C ABI (include/fgw_kv.h)
// on the current stream of the tensors' device. As in launch_shim.cpp the C entry points are not
// linked: bind() takes their addresses from the library that fgw_amd._lib loaded. Host code only.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <map>
#include <numeric>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/fgw_kv.h"

namespace {

struct Entries {
  decltype(&fgw_kv_last_error) last_error;
  decltype(&fgw_rotary_apply) rotary_apply;
  decltype(&fgw_kv_append) append;
  decltype(&fgw_kv_extend_workspace) extend_workspace;
  decltype(&fgw_kv_extend) extend;
  decltype(&fgw_pages_workspace) pages_workspace;
  decltype(&fgw_pages_reserve) reserve;
  decltype(&fgw_pages_fork) fork;
  decltype(&fgw_pages_free) free_rows;
  decltype(&fgw_pages_compact) compact;
  decltype(&fgw_pages_copy) copy;
} entries = {};

struct Refused : std::runtime_error {  // ValueError
  using std::runtime_error::runtime_error;
};
struct WrongType : std::runtime_error {  // TypeError
  using std::runtime_error::runtime_error;
};

void need(bool ok, const char* message) {
  if (!ok) throw Refused(message);
}

void check(int rc) {
  if (rc == FGW_MHA_OK) return;
  const std::string message = entries.last_error();
  if (rc == FGW_MHA_EHIP) throw std::runtime_error(message);
  throw Refused(message);
}

struct Args {
  PyObject* const* items;
  Py_ssize_t count, at = 0;
  PyObject* next() {
    if (at >= count) throw WrongType("arguments are missing");
    return items[at++];
  }
  at::Tensor tensor() {
    PyObject* a = next();
    if (!THPVariable_Check(a)) throw WrongType("arguments must be torch tensors");
    return THPVariable_Unpack(a);
  }
  at::Tensor maybe() {  // undefined for None
    if (at < count && items[at] == Py_None) {
      ++at;
      return at::Tensor();
    }
    return tensor();
  }
  int64_t integer() {
    const long long x = PyLong_AsLongLong(next());
    if (x == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      throw WrongType("an integer is required");
    }
    return x;
  }
  int32_t int32() {
    const int64_t x = integer();
    need(x >= INT32_MIN && x <= INT32_MAX, "an integer does not fit in 32 bits");
    return (int32_t)x;
  }
  double real() {
    const double x = PyFloat_AsDouble(next());
    if (x == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      throw WrongType("a number is required");
    }
    return x;
  }
};

template <PyObject* (*F)(Args&)>
PyObject* guarded(PyObject*, PyObject* const* items, Py_ssize_t count) {
  try {
    Args args{items, count};
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const WrongType& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

const char* kSameGpu = "contiguous inputs on the same GPU required";

void on(const at::Tensor& x, const c10::Device& device) {
  need(x.device() == device && device.is_cuda(), kSameGpu);
}

// int32 metadata of the given sizes (-1: any), contiguous on the device.
const int32_t* metadata(const at::Tensor& x, std::initializer_list<int64_t> sizes,
                        const c10::Device& device, const char* shape_message = "metadata shape mismatch") {
  need(x.scalar_type() == at::kInt, "int32 metadata required");
  need(x.dim() == (int64_t)sizes.size(), shape_message);
  int i = 0;
  for (int64_t n : sizes) {
    need(n < 0 || x.size(i) == n, shape_message);
    ++i;
  }
  on(x, device);
  need(x.is_contiguous(), kSameGpu);
  return static_cast<const int32_t*>(x.data_ptr());
}

int32_t size32(int64_t n) {
  need(n <= INT32_MAX, "an extent does not fit in 32 bits");
  return (int32_t)n;
}

// Rows [T, H, D] whose last dim is contiguous.
fgw_kv_rows rows(const at::Tensor& x, const c10::Device& device) {
  need(x.dim() == 3 && x.size(1) > 0 && x.size(2) > 0, "expected rows [T, H, D]");
  on(x, device);
  need(x.size(0) == 0 || x.stride(2) == 1, "the last dim of the rows must be contiguous");
  // Strides along dims of one element are never walked.
  const int64_t t = x.size(0) > 1 ? x.stride(0) : 0, h = x.size(1) > 1 ? x.stride(1) : 0;
  need(t >= 0 && h >= 0, "negative strides");
  return fgw_kv_rows{x.data_ptr(), t, h};
}

bool same_sizes(const at::Tensor& a, const at::Tensor& b) { return a.sizes() == b.sizes(); }

// First byte of a tensor without negative strides, and the byte behind its last one (empty: none).
std::pair<const char*, const char*> extent(const at::Tensor& x) {
  if (x.numel() == 0) return {nullptr, nullptr};
  const char* first = static_cast<const char*>(x.data_ptr());
  int64_t last = 0;
  for (int64_t i = 0; i < x.dim(); ++i) last += (x.size(i) - 1) * x.stride(i);
  return {first, first + (last + 1) * (int64_t)x.element_size()};
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const auto x = extent(a), y = extent(b);
  return x.first < y.second && y.first < x.second;
}
// Whether two tensors without negative strides share memory; true where that is not ruled out. Views
// of one buffer lie in each other's range without that: heads side by side in every token, or the
// parts of a [T, H, 3, D] projection. Those are told apart modulo a length m: dims whose stride is a
// multiple of m fall away, the others span a range, and two ranges that are apart on a circle of m
// bytes are apart in memory. m is tried at every stride and at their greatest common divisor.
bool shares_memory(const at::Tensor& a, const at::Tensor& b) {
  if (!overlap(a, b)) return false;
  const int64_t apart = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  auto stride = [](const at::Tensor& x, int64_t i) { return x.size(i) > 1 ? x.stride(i) * (int64_t)x.element_size() : 0; };
  auto disjoint = [&](int64_t m) {
    auto span = [&](const at::Tensor& x) {
      int64_t bytes = x.element_size();
      for (int64_t i = 0; i < x.dim(); ++i) bytes += stride(x, i) % m ? (x.size(i) - 1) * stride(x, i) : 0;
      return bytes;
    };
    const int64_t at = (apart % m + m) % m;  // of b's range behind the start of a's
    return at >= span(a) && at + span(b) <= m;
  };
  int64_t common = 0;
  for (const at::Tensor* x : {&a, &b})
    for (int64_t i = 0; i + 1 < x->dim(); ++i) {
      const int64_t m = stride(*x, i);
      if (m > 0 && disjoint(m)) return false;
      common = std::gcd(common, m);
    }
  return common == 0 || !disjoint(common);
}

// What a call writes shares no memory with what it reads (undefined tensors: not given).
typedef std::initializer_list<const at::Tensor*> Tensors;
void apart(Tensors written, Tensors read, const char* message) {
  std::pair<const char*, const char*> spans[4] = {};
  size_t n = 0;
  for (const at::Tensor* w : written) {
    if (w->defined()) spans[n] = extent(*w);
    ++n;
  }
  for (const at::Tensor* r : read) {
    if (!r->defined()) continue;
    const auto x = extent(*r);
    n = 0;
    for (const at::Tensor* w : written) {
      const auto& y = spans[n++];
      need(!(x.first < y.second && y.first < x.second) || !shares_memory(*w, *r), message);
    }
  }
}

// An output given by the caller: no two of its rows share memory, and it is `from` itself or has
// memory apart from it.
void check_out(const at::Tensor& out, const at::Tensor& from) {
  need(same_sizes(out, from) && out.scalar_type() == from.scalar_type(), "out does not match the rows");
  need(out.dim() == 3 && out.stride(0) >= 0 && out.stride(1) >= 0, "negative strides");
  need(!shares_memory(out, from) || (out.data_ptr() == from.data_ptr() && out.strides() == from.strides()),
       "out must be the rows themselves or memory apart from them");
  const int64_t span = out.size(2);
  need(out.numel() == 0 || out.size(1) == 1 || out.stride(1) >= span, "the rows of out overlap");
  need(out.numel() == 0 || out.size(0) == 1 ||
           out.stride(0) >= (out.size(1) - 1) * (out.size(1) > 1 ? out.stride(1) : 0) + span ||
           (out.size(1) > 1 && out.stride(1) >= (out.size(0) - 1) * out.stride(0) + span),
       "the rows of out overlap");
}

// A call has written to these tensors of its caller: their version moves, as after any operation in
// place, so that a gradient that has saved what they held before is refused and not computed from
// what they hold now (inference tensors have no version).
void changed(Tensors written) {
  for (const at::Tensor* x : written)
    if (x->defined() && !x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
}

// Calls that write to tensors of their caller record no gradient: none of those may require one while
// gradients are recorded, or have a tangent of forward mode.
void writable(Tensors written) {
  for (const at::Tensor* x : written)
    need(!x->defined() || !x->_fw_grad(0).defined(), "a tensor that the call writes has a forward gradient, which is not recorded");
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* x : written)
    need(!x->defined() || !x->requires_grad(), "a tensor that the call writes requires a gradient, which is not recorded");
}

hipStream_t stream_of(const c10::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

void positions_of(const at::Tensor& x, int64_t tokens, const c10::Device& device, const void*& data,
                  int32_t& wide) {
  need(x.scalar_type() == at::kInt || x.scalar_type() == at::kLong, "int32 or int64 positions required");
  need(x.dim() == 1 && x.size(0) == tokens, "positions must be [T]");
  on(x, device);
  need(x.is_contiguous(), kSameGpu);
  data = x.data_ptr();
  wide = x.scalar_type() == at::kLong;
}

fgw_kv_rotary rotary_of(Args& a, const c10::Device& device) {
  const at::Tensor turns = a.maybe();
  fgw_kv_rotary r = {};
  r.dim = a.int32();
  r.interleaved = a.int32();
  r.scale = (float)a.real();
  if (turns.defined()) {
    need(turns.scalar_type() == at::kLong && turns.dim() == 1 && turns.is_contiguous() &&
             2 * turns.size(0) == r.dim, "rotary frequencies must be int64 [dim / 2]");
    need(turns.device() == device, "the rotary frequencies must be on the GPU of the rows");
    r.turns = static_cast<const uint64_t*>(turns.data_ptr());
  }
  return r;
}

// (x, positions, turns, rot, interleaved, scale, inverse, out | None) -> out
PyObject* rotate(Args& a) {
  const at::Tensor x = a.tensor(), positions = a.tensor();
  const c10::Device device = x.device();
  need(device.is_cuda(), "rows must be on a GPU");
  fgw_rotary_args r = {};
  r.rotary = rotary_of(a, device);
  r.rotary.inverse = a.int32();
  at::Tensor out = a.maybe();
  r.x = rows(x, device);
  switch (x.scalar_type()) {
    case at::kHalf: r.dtype = FGW_KV_FLOAT16; break;
    case at::kBFloat16: r.dtype = FGW_KV_BFLOAT16; break;
    case at::kFloat: r.dtype = FGW_KV_FLOAT32; break;
    default: throw Refused("FP16, BF16 or FP32 rows required");
  }
  r.tokens = size32(x.size(0));
  r.heads = size32(x.size(1));
  r.dim = size32(x.size(2));
  positions_of(positions, x.size(0), device, r.positions, r.positions64);
  const c10::DeviceGuard guard(device);
  const at::Tensor given = out;
  writable({&given});
  if (out.defined()) {
    check_out(out, x);
    apart({&out}, {&positions}, "out must not share memory with the positions");
  } else {
    out = at::empty(x.sizes(), x.options());
  }
  r.out = rows(out, device);
  check(entries.rotary_apply(&r, stream_of(device)));
  changed({&given});
  return THPVariable_Wrap(std::move(out));
}

int32_t cache_dtype(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  need((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) &&
           k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
       "matching FP16/BF16 Q/K/V required");
  return q.scalar_type() == at::kHalf ? FGW_KV_FLOAT16 : FGW_KV_BFLOAT16;
}

void check_pool(const at::Tensor& k, const at::Tensor& v, int64_t dim, const c10::Device& device) {
  need(k.dim() == 3 && same_sizes(k, v), "K/V shape mismatch");
  need(k.size(2) == dim && k.size(1) > 0, "K/V shape mismatch");
  on(k, device);
  on(v, device);
  need(k.is_contiguous() && v.is_contiguous(), kSameGpu);
}

// (q, k, v, k_cache, v_cache, table, lens, cu, page, turns | None, rot, interleaved, scale,
//  positions | None, q_out | None) -> q_out
PyObject* append(Args& a) {
  const at::Tensor q = a.tensor(), k = a.tensor(), v = a.tensor(), kc = a.tensor(), vc = a.tensor();
  const at::Tensor table = a.tensor(), lens = a.tensor(), cu = a.tensor();
  const c10::Device device = q.device();
  need(device.is_cuda(), kSameGpu);
  fgw_kv_append_args r = {};
  r.page_size = a.int32();
  r.rotary = rotary_of(a, device);
  const at::Tensor positions = a.maybe();
  at::Tensor q_out = a.maybe();
  r.q = rows(q, device);
  r.k = rows(k, device);
  r.v = rows(v, device);
  r.dtype = cache_dtype(q, k, v);
  need(kc.scalar_type() == q.scalar_type() && vc.scalar_type() == q.scalar_type(),
       "matching FP16/BF16 Q/K/V required");
  need(same_sizes(k, v) && k.size(0) == q.size(0) && k.size(2) == q.size(2), "K/V shape mismatch");
  check_pool(kc, vc, q.size(2), device);
  need(kc.size(1) == k.size(1), "K/V shape mismatch");
  need(!overlap(kc, vc), "the K and V pools must be apart from each other");
  need(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0,
       "positive Q extents and rank-2 table required");
  const int64_t batch = table.size(0);
  r.block_table = metadata(table, {batch, -1}, device);
  r.cache_seqlens = metadata(lens, {batch}, device);
  r.cu_seqlens = metadata(cu, {batch + 1}, device);
  r.k_cache = kc.data_ptr();
  r.v_cache = vc.data_ptr();
  r.pool_rows = kc.size(0);
  r.tokens = size32(q.size(0));
  r.batch = size32(batch);
  r.heads = size32(q.size(1));
  r.kv_heads = size32(k.size(1));
  r.dim = size32(q.size(2));
  r.width = size32(table.size(1));
  if (positions.defined()) positions_of(positions, q.size(0), device, r.positions, r.positions64);
  const c10::DeviceGuard guard(device);
  // (Another thread's rows may be read after this one's are written.)
  const char* const message = "q_out and the pools must not share memory with what the call reads";
  apart({&kc, &vc}, {&q, &q_out}, message);
  apart({&kc, &vc, &q_out}, {&k, &v, &table, &lens, &cu, &positions}, message);
  const at::Tensor given = q_out;
  writable({&kc, &vc, &given});
  if (q_out.defined())
    check_out(q_out, q);
  else
    q_out = at::empty(q.sizes(), q.options());
  r.q_out = rows(q_out, device);
  check(entries.append(&r, stream_of(device)));
  changed({&kc, &vc, &given});
  return THPVariable_Wrap(std::move(q_out));
}

// Arrival counters of the fused joins: one zeroed buffer per (device, stream), grown as calls need
// more. Every call leaves its counters at zero, so calls in stream order share them; calls on other
// streams have their own. A captured call takes none (its replays may run on any stream): its
// tiles are joined by a second launch, with the same arithmetic. Buffers live until the process
// ends, replaced ones too, since a kernel in flight may count in them.
int32_t* arrival_counters(const c10::Device& device, hipStream_t stream, int64_t need) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess || status != hipStreamCaptureStatusNone)
    return nullptr;
  static auto* buffers = new std::map<std::pair<int, uintptr_t>, at::Tensor>();
  static auto* retired = new std::vector<at::Tensor>();
  at::Tensor& buffer = (*buffers)[{device.index(), reinterpret_cast<uintptr_t>(stream)}];
  if (!buffer.defined() || buffer.numel() < need) {
    if (buffer.defined()) retired->push_back(buffer);
    buffer = at::zeros({need}, at::TensorOptions().device(device).dtype(at::kInt));
  }
  return static_cast<int32_t*>(buffer.data_ptr());
}

// (q, k_cache, v_cache, table, lens, cu, max_new, page, heads, kv_heads, dim, bf16, device, causal,
//  window, scale, num_cus, out | None) -> out
PyObject* extend(Args& a) {
  const at::Tensor q = a.tensor(), kc = a.tensor(), vc = a.tensor();
  const at::Tensor table = a.tensor(), lens = a.tensor(), cu = a.tensor();
  fgw_kv_extend_args r = {};
  r.max_new = a.int32();
  r.page_size = a.int32();
  r.heads = a.int32();
  r.kv_heads = a.int32();
  r.dim = a.int32();
  const bool bf16 = a.int32() != 0;
  const c10::Device device(c10::kCUDA, (c10::DeviceIndex)a.int32());
  r.causal = a.int32();
  r.window = a.int32();
  r.scale = (float)a.real();
  r.num_cus = a.int32();
  at::Tensor out = a.maybe();
  r.q = rows(q, device);
  need(q.size(1) == r.heads && q.size(2) == r.dim, "tensor shapes do not match the built kernel");
  r.dtype = cache_dtype(q, kc, vc);
  need((r.dtype == FGW_KV_BFLOAT16) == bf16, "matching FP16/BF16 Q/K/V required");
  check_pool(kc, vc, r.dim, device);
  need(kc.size(1) == r.kv_heads, "tensor shapes do not match the built kernel");
  need(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0,
       "positive Q extents and rank-2 table required");
  const int64_t batch = table.size(0);
  r.block_table = metadata(table, {batch, -1}, device);
  r.cache_seqlens = metadata(lens, {batch}, device);
  r.cu_seqlens = metadata(cu, {batch + 1}, device);
  r.k_cache = kc.data_ptr();
  r.v_cache = vc.data_ptr();
  r.pool_rows = kc.size(0);
  r.tokens = size32(q.size(0));
  r.batch = size32(batch);
  r.width = size32(table.size(1));
  need(r.max_new > 0, "max_new must be positive");
  int64_t floats = 0, counters = 0;
  check(entries.extend_workspace(&r, &floats, &counters));
  const c10::DeviceGuard guard(device);
  const at::Tensor given = out;
  writable({&given});
  if (out.defined()) {
    need(same_sizes(out, q) && out.scalar_type() == q.scalar_type(), "out does not match the rows");
    on(out, device);
    need(out.is_contiguous(), kSameGpu);
    need(!shares_memory(out, q), "out must not be q or share memory with it");
    apart({&out}, {&kc, &vc, &table, &lens, &cu}, "out must not share memory with what the call reads");
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  r.out = out.data_ptr();
  at::Tensor work;
  if (floats > 0) {
    work = at::empty({floats}, q.options().dtype(at::kFloat));
    r.workspace = static_cast<float*>(work.data_ptr());
  }
  const hipStream_t stream = stream_of(device);
  if (counters > 0) r.counters = arrival_counters(device, stream, counters);
  check(entries.extend(&r, stream));
  changed({&given});
  return THPVariable_Wrap(std::move(out));
}

// refs, table, lens, page_size of a call, and the lists that it reads while the books change.
fgw_pages_books books_of(const at::Tensor& refs, const at::Tensor& table, const at::Tensor& lens,
                         int32_t page, Tensors lists) {
  const c10::Device device = refs.device();
  need(device.is_cuda(), kSameGpu);
  need(refs.dim() == 1 && table.dim() == 2 && lens.dim() == 1 && refs.size(0) > 0 && table.size(0) > 0 &&
           table.size(1) > 0, "expected refs [pages], table [rows, width] and lens [rows]");
  fgw_pages_books b;
  b.refs = const_cast<int32_t*>(metadata(refs, {-1}, device));
  b.table = const_cast<int32_t*>(metadata(table, {-1, -1}, device));
  b.lens = const_cast<int32_t*>(metadata(lens, {table.size(0)}, device));
  b.pages = size32(refs.size(0));
  b.rows = size32(table.size(0));
  b.width = size32(table.size(1));
  b.page_size = page;
  const char* const message = "refs, table and lens must not share memory with each other or with what the call reads";
  apart({&refs, &table, &lens}, lists, message);
  apart({&refs}, {&table, &lens}, message);
  apart({&table}, {&lens}, message);
  return b;
}

struct PoolList {
  std::vector<void*> data;
  std::vector<int64_t> bytes;
  std::vector<at::Tensor> tensors;
  void changed() const {
    for (const at::Tensor& x : tensors) ::changed({&x});
  }
  fgw_pages_pools view() const { return {data.data(), bytes.data(), (int32_t)data.size()}; }
};

// A tuple or list of pools [pages * page_size, ...], contiguous on the device: each apart from the
// lists and books of the call, and from the others (but for one given twice, which is copied twice
// to the same contents).
PoolList pools_of(PyObject* seq, int64_t pages, int32_t page, const c10::Device& device, Tensors others) {
  if (!PyTuple_Check(seq) && !PyList_Check(seq)) throw WrongType("pools must be a list or a tuple of tensors");
  PoolList list;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(item)) throw WrongType("pools must be a list or a tuple of tensors");
    const at::Tensor& x = THPVariable_Unpack(item);
    writable({&x});
    on(x, device);
    need(x.is_contiguous(), kSameGpu);
    need(page > 0 && x.dim() >= 1 && x.size(0) == pages * page, "a pool must have pages * page_size rows");
    list.data.push_back(x.data_ptr());
    list.bytes.push_back(x.numel() / pages * x.element_size());
    list.tensors.push_back(x);
    apart({&x}, others, "pools must not share memory with the books or lists of the call");
  }
  std::vector<std::pair<const char*, int64_t>> spans;
  for (const at::Tensor& x : list.tensors) spans.emplace_back(static_cast<const char*>(x.data_ptr()), (int64_t)x.nbytes());
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    need(spans[i - 1].first + spans[i - 1].second <= spans[i].first || spans[i - 1] == spans[i],
         "pools must not share memory with each other");
  return list;
}

at::Tensor ints(int64_t n, const c10::Device& device) {
  return at::empty({n}, at::TensorOptions().device(device).dtype(at::kInt));
}
int32_t* ptr(const at::Tensor& x) { return static_cast<int32_t*>(x.data_ptr()); }

// (refs, table, lens, counts, page) -> status
PyObject* reserve(Args& a) {
  const at::Tensor refs = a.tensor(), table = a.tensor(), lens = a.tensor(), counts = a.tensor();
  const fgw_pages_books b = books_of(refs, table, lens, a.int32(), {});
  // (The lengths themselves may be the counts: a row's are read before they change.)
  const char* const message = "counts must not share memory with the books";
  apart({&refs, &table}, {&counts}, message);
  if (counts.data_ptr() != lens.data_ptr()) apart({&lens}, {&counts}, message);
  const c10::Device device = refs.device();
  const int32_t* c = metadata(counts, {b.rows}, device);
  const c10::DeviceGuard guard(device);
  at::Tensor status = ints(2, device), work = ints(entries.pages_workspace(b.pages, b.rows), device);
  check(entries.reserve(&b, c, ptr(status), ptr(work), stream_of(device)));
  changed({&refs, &table, &lens});
  return THPVariable_Wrap(std::move(status));
}

// (pools, refs, table, lens, parents, children, page) -> status
PyObject* fork_rows(Args& a) {
  PyObject* list = a.next();
  const at::Tensor refs = a.tensor(), table = a.tensor(), lens = a.tensor();
  const at::Tensor parents = a.tensor(), children = a.tensor();
  const fgw_pages_books b = books_of(refs, table, lens, a.int32(), {&parents, &children});
  const c10::Device device = refs.device();
  const PoolList pools = pools_of(list, b.pages, b.page_size, device, {&refs, &table, &lens, &parents, &children});
  const int32_t* p = metadata(parents, {-1}, device);
  const int32_t* c = metadata(children, {parents.size(0)}, device);
  const int32_t pairs = size32(parents.size(0));
  const c10::DeviceGuard guard(device);
  at::Tensor status = ints(2, device), work = ints(entries.pages_workspace(b.pages, pairs), device);
  const fgw_pages_pools view = pools.view();
  check(entries.fork(&b, &view, p, c, pairs, ptr(status), ptr(work), stream_of(device)));
  changed({&refs, &table, &lens});
  pools.changed();
  return THPVariable_Wrap(std::move(status));
}

// (refs, table, lens, rows, page)
PyObject* free_rows(Args& a) {
  const at::Tensor refs = a.tensor(), table = a.tensor(), lens = a.tensor(), rows = a.tensor();
  const fgw_pages_books b = books_of(refs, table, lens, a.int32(), {&rows});
  const c10::Device device = refs.device();
  const int32_t* r = metadata(rows, {-1}, device);
  const c10::DeviceGuard guard(device);
  check(entries.free_rows(&b, r, size32(rows.size(0)), stream_of(device)));
  changed({&refs, &table, &lens});
  Py_RETURN_NONE;
}

// (pools, refs, table, lens, page) -> moved
PyObject* compact(Args& a) {
  PyObject* list = a.next();
  const at::Tensor refs = a.tensor(), table = a.tensor(), lens = a.tensor();
  const fgw_pages_books b = books_of(refs, table, lens, a.int32(), {});
  const c10::Device device = refs.device();
  const PoolList pools = pools_of(list, b.pages, b.page_size, device, {&refs, &table, &lens});
  const c10::DeviceGuard guard(device);
  at::Tensor moved = ints(1, device), work = ints(entries.pages_workspace(b.pages, 0), device);
  const fgw_pages_pools view = pools.view();
  check(entries.compact(&b, &view, ptr(moved), ptr(work), stream_of(device)));
  changed({&refs, &table, &lens});
  pools.changed();
  return THPVariable_Wrap(std::move(moved));
}

// (pools, src, dst, pages, page)
PyObject* copy_pages(Args& a) {
  PyObject* list = a.next();
  const at::Tensor src = a.tensor(), dst = a.tensor();
  const int32_t pages = a.int32(), page = a.int32();
  const c10::Device device = src.device();
  need(device.is_cuda(), kSameGpu);
  need(pages > 0, "positive pages required");
  const PoolList pools = pools_of(list, pages, page, device, {&src, &dst});
  const int32_t* s = metadata(src, {-1}, device);
  const int32_t* d = metadata(dst, {src.size(0)}, device);
  const c10::DeviceGuard guard(device);
  const fgw_pages_pools view = pools.view();
  check(entries.copy(&view, pages, s, d, size32(src.size(0)), stream_of(device)));
  pools.changed();
  Py_RETURN_NONE;
}

// x -> bool: x is a dual tensor of forward-mode derivatives.
PyObject* has_tangent(Args& a) { return PyBool_FromLong(a.tensor()._fw_grad(0).defined()); }

// (a, b) -> bool: what the calls take for sharing memory, on any device.
PyObject* shares_memory_of(Args& a) {
  const at::Tensor x = a.tensor(), y = a.tensor();
  return PyBool_FromLong(shares_memory(x, y));
}

// The addresses of the C entry points, in the order of Entries.
PyObject* bind(Args& a) {
  void** const table = reinterpret_cast<void**>(&entries);
  constexpr size_t n = sizeof(Entries) / sizeof(void*);
  void* found[n];
  for (size_t i = 0; i < n; ++i) {
    found[i] = PyLong_AsVoidPtr(a.next());
    if (!found[i]) {
      PyErr_Clear();
      throw WrongType("addresses of the C entry points required");
    }
  }
  for (size_t i = 0; i < n; ++i) table[i] = found[i];
  Py_RETURN_NONE;
}

#define FGW_FAST(F) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&guarded<F>))
PyMethodDef methods[] = {
    {"bind", FGW_FAST(bind), METH_FASTCALL, "addresses of the C entry points"},
    {"rotate", FGW_FAST(rotate), METH_FASTCALL, "fgw_rotary_apply"},
    {"append", FGW_FAST(append), METH_FASTCALL, "fgw_kv_append"},
    {"extend", FGW_FAST(extend), METH_FASTCALL, "fgw_kv_extend"},
    {"reserve", FGW_FAST(reserve), METH_FASTCALL, "fgw_pages_reserve"},
    {"fork", FGW_FAST(fork_rows), METH_FASTCALL, "fgw_pages_fork"},
    {"free", FGW_FAST(free_rows), METH_FASTCALL, "fgw_pages_free"},
    {"compact", FGW_FAST(compact), METH_FASTCALL, "fgw_pages_compact"},
    {"copy", FGW_FAST(copy_pages), METH_FASTCALL, "fgw_pages_copy"},
    {"has_tangent", FGW_FAST(has_tangent), METH_FASTCALL, "whether a tensor has a forward gradient"},
    {"shares_memory", FGW_FAST(shares_memory_of), METH_FASTCALL, "whether two tensors may share memory"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_kv", "C++ calls over the fgw_kv C ABI", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__kv(void) { return PyModule_Create(&module_def); }
