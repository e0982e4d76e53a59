// Host side of the paged-cache operators: argument checks, outputs, scratch
// and the launch, from torch tensors.
//
// The other operators fill their launch blocks in Python through ctypes,
// which a message of many layers pays once.  These are called once a layer
// and decode step on a few rows, where that took 27 us (append) and 29
// (attention) against 3 to 9 us of kernel; here it is 6 and 7.  What is
// refused is refused as TypeError (a dtype, a rank) or ValueError (a size, a
// stride, a place, a gradient).
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/util/SmallVector.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>

#include "../kvs_types.h"

using at::Tensor;
using std::optional;

extern "C" {
int kvs_append_kv(const kvs::AppendLaunch* L, void* stream);
int kvs_read_kv4(const kvs::Read4Launch* L, void* stream);
int kvs_append_kv8(const kvs::AppendLaunch* L, void* stream);
int kvs_read_kv8(const kvs::Read4Launch* L, void* stream);
long long kvs_attn4_scratch_bytes(const kvs::Attn4Launch* L);
int kvs_attention_kv4(const kvs::Attn4Launch* L, void* stream);
long long kvs_attn8_scratch_bytes(const kvs::Attn4Launch* L);
int kvs_attention_kv8(const kvs::Attn4Launch* L, void* stream);
const char* kvs_last_error_string(void);
}

namespace {

constexpr int64_t kDim = kvs::kHeadDim;
constexpr int kMaxDevices = 64;
uint32_t* g_err[kMaxDevices] = {};  // device error words, set once a device

// Thrown before any work when a device's error word is not known yet.
struct NoErrorWord : std::runtime_error {
  using std::runtime_error::runtime_error;
};

bool half_type(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

void check_heads(const char* name, const Tensor& t, at::ScalarType dt) {
  TORCH_CHECK_TYPE(half_type(t) && t.scalar_type() == dt, name,
                   " must be bf16 or fp16, one dtype for all, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == kDim, name, " must be [tokens, heads, 128], got ",
                    t.sizes());
}

bool rows_ok(const Tensor& t) {
  return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned16(t);
}
// The rows as the kernels read them: copied only when they are not aligned.
Tensor rows(const Tensor& t) { return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

Tensor index(const char* name, const Tensor& t) {
  TORCH_CHECK_TYPE(
      (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1, name,
      " must be a one-dimensional int32 or int64 tensor");
  return t.contiguous();
}

// What is written has each element once: every stride goes past all that is inside it.
void check_distinct(const char* name, const Tensor& t) {
  c10::SmallVector<int64_t, 8> dims;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.push_back(d);
  std::sort(dims.begin(), dims.end(),
            [&](int64_t a, int64_t b) { return t.stride(a) < t.stride(b); });
  int64_t extent = 1;
  for (const int64_t d : dims) {
    TORCH_CHECK_VALUE(t.numel() == 0 || t.stride(d) >= extent, name,
                      " is written and must not overlap itself, got strides ", t.strides());
    extent += (t.size(d) - 1) * t.stride(d);
  }
}
void check_out(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes(), name,
                    " must match the query's shape and dtype");
  TORCH_CHECK_VALUE(rows_ok(t), name, " must have 16-byte aligned rows");
  check_distinct(name, t);
  TORCH_CHECK_VALUE(at::get_overlap_status(t, like) != at::MemOverlapStatus::Partial, name,
                    " overlaps the query without being it");
}

int groups4(const Tensor& cache) {
  TORCH_CHECK_TYPE(cache.scalar_type() == at::kByte && cache.dim() == 4,
                   "a 4-bit cache is a uint8 [blocks, heads, block_size, row_bytes] tensor");
  const int64_t rb = cache.size(3), bs = cache.size(2);
  TORCH_CHECK_VALUE(rb == 136 || rb == 144 || rb == 160,
                    "a 4-bit cache's row has 136, 144 or 160 bytes, got ", rb);
  TORCH_CHECK_VALUE(bs > 0 && bs % 16 == 0, "block_size must be a multiple of 16");
  TORCH_CHECK_VALUE(cache.stride(3) == 1 && cache.stride(2) == rb && cache.stride(0) % 16 == 0 &&
                        cache.stride(1) % 16 == 0 && aligned16(cache),
                    "a 4-bit cache's records must be contiguous and 16-byte aligned, got strides ",
                    cache.strides());
  TORCH_CHECK_VALUE(cache.size(0) < (1ll << 31) && bs < (1 << 20) && cache.stride(0) >= 0 &&
                        cache.stride(0) < (1ll << 32),
                    "a 4-bit cache has at most 2^31 blocks, 4 GB apart");
  return static_cast<int>((rb - 128) / 8);
}

// Whether a cache is one of 8 bits; the other uint8 caches are taken for 4-bit ones.
bool is_kv8(const Tensor& cache) {
  return cache.scalar_type() == at::kByte && cache.dim() == 4 && cache.size(3) == kDim;
}
// The block size of an 8-bit cache.
int64_t block8(const Tensor& cache) {
  TORCH_CHECK_TYPE(cache.scalar_type() == at::kByte && cache.dim() == 4,
                   "an 8-bit cache is a uint8 [blocks, heads, 2 * block_size + 1, 128] tensor");
  const int64_t rows = cache.size(2), bs = (rows - 1) / 2;
  TORCH_CHECK_VALUE(cache.size(3) == kDim && rows % 2 == 1 && bs > 0 && bs % 16 == 0 && bs <= 1024,
                    "an 8-bit cache is [blocks, heads, 2 * block_size + 1, 128] with a block_size "
                    "that is a multiple of 16 up to 1024, got ", cache.sizes());
  TORCH_CHECK_VALUE(cache.stride(3) == 1 && cache.stride(2) == kDim && cache.stride(0) % 16 == 0 &&
                        cache.stride(1) % 16 == 0 && aligned16(cache),
                    "an 8-bit cache's records must be contiguous and 16-byte aligned, got strides ",
                    cache.strides());
  for (int d = 0; d < 2; ++d)  // the copy engine's limits
    TORCH_CHECK_VALUE(cache.size(d) < (1ll << 31) &&
                          (cache.size(d) <= 1 ||
                           (cache.stride(d) > 0 && cache.stride(d) < (1ll << 40))),
                      "an 8-bit cache's records do not overlap and are at most 2^40 bytes apart, "
                      "got strides ", cache.strides());
  return bs;
}

void on_device(const char* what, const at::Device& dev, std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK_VALUE(dev.is_cuda(), what, " needs CUDA tensors");
  for (const Tensor* t : ts)
    TORCH_CHECK_VALUE(t == nullptr || t->device() == dev, what, ": tensors on ", t->device(),
                      " and ", dev);
  TORCH_CHECK_VALUE(dev.index() < kMaxDevices, what, ": device index too large");
  if (g_err[dev.index()] == nullptr) throw NoErrorWord("no error word");
}
// There is no backward pass: a gradient would be lost without a word.
void no_gradient(const char* what, std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_VALUE(t == nullptr || !t->requires_grad(), what,
                      " has no backward pass: call it under torch.no_grad() or on detached tensors");
}
const Tensor* opt(const optional<Tensor>& t) { return t.has_value() ? &*t : nullptr; }

void launched(int rc, const char* what) {
  TORCH_CHECK(rc != -2, what, ": the call is too large for one launch");
  TORCH_CHECK(rc != -3, what, ": the driver makes no tensor map of this cache");
  TORCH_CHECK(rc == 0, what, " failed: ", kvs_last_error_string());
}

int int_of(const char* what, int64_t n) {
  TORCH_CHECK_VALUE(n >= 0 && n < (1ll << 31), what, " is too large: ", n);
  return static_cast<int>(n);
}

optional<Tensor> append_kv(const Tensor& cache, const Tensor& key_in, const Tensor& value_in,
                           const Tensor& slot_mapping, const optional<Tensor>& positions,
                           const optional<Tensor>& cos_sin, const optional<Tensor>& query,
                           bool interleaved, optional<Tensor> query_out) {
  const at::ScalarType dt = key_in.scalar_type();
  check_heads("key", key_in, dt);
  check_heads("value", value_in, dt);
  TORCH_CHECK_VALUE(value_in.sizes() == key_in.sizes(), "key ", key_in.sizes(), " and value ",
                    value_in.sizes(), " differ");
  const at::Device dev = key_in.device();
  const Tensor slots = index("slot_mapping", slot_mapping);
  const int64_t T = key_in.size(0), H = key_in.size(1), n = slots.size(0);
  TORCH_CHECK_VALUE(n <= T, n, " slots for ", T, " tokens");
  kvs::AppendLaunch L = {};
  int64_t nb, bs, hc;
  const bool eight = is_kv8(cache);
  if (eight) {
    bs = block8(cache), nb = cache.size(0), hc = cache.size(1);
    L.block_stride = cache.stride(0), L.head_stride = cache.stride(1);
  } else if (cache.scalar_type() == at::kByte) {
    L.groups = groups4(cache);
    nb = cache.size(0), hc = cache.size(1), bs = cache.size(2);
    L.block_stride = cache.stride(0), L.head_stride = cache.stride(1);
  } else {
    TORCH_CHECK_TYPE(cache.scalar_type() == dt, "cache is ", cache.scalar_type(), ", keys are ",
                     dt);
    TORCH_CHECK_VALUE(cache.dim() == 5 && cache.size(4) == kDim &&
                          (cache.size(0) == 2 || cache.size(1) == 2),
                      "expected a [2, nb, bs, H, 128] layer, got ", cache.sizes());
    TORCH_CHECK_VALUE(cache.stride(4) == 1 && cache.stride(0) % 8 == 0 &&
                          cache.stride(1) % 8 == 0 && cache.stride(2) % 8 == 0 &&
                          cache.stride(3) % 8 == 0 && aligned16(cache),
                      "the cache's rows must be 16-byte aligned, got strides ", cache.strides());
    const int plane = cache.size(1) == 2 && cache.size(0) != 2 ? 1 : 0;
    L.kv_stride = cache.stride(plane), L.block_stride = cache.stride(1 - plane);
    nb = cache.size(1 - plane), bs = cache.size(2), hc = cache.size(3);
    L.slot_stride = cache.stride(2), L.head_stride = cache.stride(3);
  }
  TORCH_CHECK_VALUE(hc == H, "the cache has ", hc, " heads, the keys ", H);
  check_distinct("cache", cache);
  L.num_slots = nb * bs, L.block_size = int_of("block_size", bs);
  const Tensor key = rows(key_in), value = rows(value_in);
  L.key = key.data_ptr(), L.value = value.data_ptr(), L.slots = slots.data_ptr();
  L.cache = cache.data_ptr();
  L.key_ts = key.stride(0), L.key_hs = key.stride(1);
  L.val_ts = value.stride(0), L.val_hs = value.stride(1);
  L.tokens = int_of("tokens", n), L.heads = int_of("heads", H);
  L.fp16 = dt == at::kHalf, L.slots64 = slots.scalar_type() == at::kLong;
  TORCH_CHECK_VALUE(positions.has_value() == cos_sin.has_value(),
                    "positions and cos_sin go together");
  TORCH_CHECK_VALUE(positions.has_value() || !query.has_value(),
                    "query is only taken to be rotated (positions and cos_sin)");
  TORCH_CHECK_VALUE(query.has_value() || !query_out.has_value(), "query_out without query");
  Tensor pos, src;
  if (positions.has_value()) {
    pos = index("positions", *positions);
    TORCH_CHECK_VALUE(pos.size(0) >= n, "positions has ", pos.size(0), " entries for ", n,
                      " tokens");
    const Tensor& t = *cos_sin;
    TORCH_CHECK_TYPE(t.dim() == 2 && (t.scalar_type() == at::kFloat || t.scalar_type() == dt),
                     "cos_sin must be [max_position, rotary_dim], fp32 or the keys' dtype");
    const int64_t rd = t.size(1);
    TORCH_CHECK_VALUE(rd > 0 && rd <= kDim && rd % 16 == 0,
                      "rotary_dim must be a multiple of 16 up to 128, got ", rd);
    TORCH_CHECK_VALUE(t.stride(1) == 1 && t.stride(0) * t.element_size() % 16 == 0 && aligned16(t),
                      "cos_sin's rows must be 16-byte aligned");
    L.pos = pos.data_ptr(), L.pos64 = pos.scalar_type() == at::kLong;
    L.table = t.data_ptr(), L.table32 = t.scalar_type() == at::kFloat;
    L.max_pos = t.size(0), L.table_stride = t.stride(0), L.rotary = static_cast<int>(rd);
    L.interleaved = interleaved;
  }
  if (query.has_value()) {
    check_heads("query", *query, dt);
    TORCH_CHECK_VALUE(query->size(0) == T, "query has ", query->size(0), " rows, key ", T);
    if (query_out.has_value()) check_out("query_out", *query_out, *query);
  }
  no_gradient("append_kv",
              {&cache, &key_in, &value_in, opt(cos_sin), opt(query), opt(query_out)});
  on_device("append_kv", dev,
            {&cache, &value_in, &slot_mapping, opt(positions), opt(cos_sin), opt(query),
             opt(query_out)});
  const c10::cuda::CUDAGuard guard(dev);
  if (query.has_value()) {
    src = rows(*query);
    if (!query_out.has_value()) {
      query_out = at::empty(query->sizes(), query->options());
      if (n < T) query_out->narrow(0, n, T - n).zero_();
    }
    L.query = src.data_ptr(), L.query_out = query_out->data_ptr();
    L.q_heads = int_of("query heads", src.size(1));
    L.q_ts = src.stride(0), L.q_hs = src.stride(1);
    L.qo_ts = query_out->stride(0), L.qo_hs = query_out->stride(1);
  }
  if (n == 0 || H + L.q_heads == 0) return query_out;
  L.err = g_err[dev.index()];
  void* const stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  launched(eight ? kvs_append_kv8(&L, stream) : kvs_append_kv(&L, stream), "append_kv");
  return query_out;
}

// Rows of a 4-bit or (EIGHT) 8-bit cache.
template <bool EIGHT>
Tensor read_rows(const Tensor& cache, const Tensor& slot_mapping, at::ScalarType dt,
                 const optional<Tensor>& out_in) {
  const char* const what = EIGHT ? "read_kv8" : "read_kv4";
  const int groups = EIGHT ? 0 : groups4(cache);
  const int64_t bs = EIGHT ? block8(cache) : cache.size(2);
  TORCH_CHECK_TYPE(dt == at::kBFloat16 || dt == at::kHalf, "dtype must be bf16 or fp16, got ", dt);
  const Tensor slots = index("slot_mapping", slot_mapping);
  const at::Device dev = cache.device();
  const int64_t nb = cache.size(0), H = cache.size(1), n = slots.size(0);
  const int64_t shape[4] = {2, n, H, kDim};
  if (out_in.has_value())
    TORCH_CHECK_VALUE(out_in->sizes() == at::IntArrayRef(shape) && out_in->scalar_type() == dt &&
                          out_in->is_contiguous() && aligned16(*out_in),
                      "out must be a contiguous ", dt, " tensor of ", at::IntArrayRef(shape));
  no_gradient(what, {opt(out_in)});
  on_device(what, dev, {&slot_mapping, opt(out_in)});
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_in.has_value() ? *out_in : at::empty(shape, cache.options().dtype(dt));
  if (n == 0 || H == 0) return out;
  kvs::Read4Launch L = {};
  L.cache = cache.data_ptr(), L.slots = slots.data_ptr(), L.out = out.data_ptr();
  L.block_stride = cache.stride(0), L.head_stride = cache.stride(1), L.num_slots = nb * bs;
  L.tokens = int_of("tokens", n), L.heads = int_of("heads", H);
  L.block_size = static_cast<int>(bs), L.groups = groups;
  L.fp16 = dt == at::kHalf, L.slots64 = slots.scalar_type() == at::kLong;
  L.err = g_err[dev.index()];
  void* const stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  launched(EIGHT ? kvs_read_kv8(&L, stream) : kvs_read_kv4(&L, stream), what);
  return out;
}

// Attention over a 4-bit or (EIGHT) 8-bit cache.
template <bool EIGHT>
std::pair<Tensor, optional<Tensor>> attention(
    const Tensor& query, const Tensor& cache, const Tensor& block_table, const Tensor& seq_lens,
    const optional<Tensor>& query_start, int64_t max_query_len, optional<double> scale,
    const optional<Tensor>& out_in, bool return_lse, bool causal) {
  const char* const what = EIGHT ? "attention_kv8" : "attention_kv4";
  check_heads("query", query, query.scalar_type());
  const int groups = EIGHT ? 0 : groups4(cache);
  const int64_t bs = EIGHT ? block8(cache) : cache.size(2);
  const at::Device dev = query.device();
  TORCH_CHECK_TYPE(block_table.scalar_type() == at::kInt && block_table.dim() == 2,
                   "block_table must be an int32 [sequences, columns] tensor");
  const int64_t R = block_table.size(0), T = query.size(0), Hq = query.size(1), H = cache.size(1);
  TORCH_CHECK_TYPE(seq_lens.scalar_type() == at::kInt && seq_lens.dim() == 1 &&
                       seq_lens.size(0) == R,
                   "seq_lens must be an int32 [", R, "] tensor");
  TORCH_CHECK_VALUE(H > 0 && Hq % H == 0, Hq, " query heads are no multiple of the cache's ", H);
  if (query_start.has_value()) {
    TORCH_CHECK_TYPE(query_start->scalar_type() == at::kInt && query_start->dim() == 1 &&
                         query_start->size(0) == R + 1,
                     "query_start must be an int32 [", R + 1, "] tensor");
    TORCH_CHECK_VALUE(max_query_len >= 1, "max_query_len must be positive");
  } else {
    TORCH_CHECK_VALUE(T >= R, T, " query rows for ", R, " sequences");
    TORCH_CHECK_VALUE(max_query_len == 1, "max_query_len needs query_start");
  }
  const double sc = scale.has_value() ? *scale : 0.08838834764831845;  // 1 / sqrt(128)
  TORCH_CHECK_VALUE(std::isfinite(sc) && sc != 0.0, "scale must be finite and not zero, got ", sc);
  if (out_in.has_value()) check_out("out", *out_in, query);
  no_gradient(what, {&query, opt(out_in)});
  on_device(what, dev,
            {&cache, &block_table, &seq_lens, opt(query_start), opt(out_in)});
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_in.has_value() ? *out_in : at::empty(query.sizes(), query.options());
  optional<Tensor> lse;
  if (return_lse) lse = at::empty({T, Hq}, query.options().dtype(at::kFloat));
  if (R == 0 || T == 0 || Hq == 0) {
    if (!out_in.has_value()) out.zero_();
    if (lse.has_value()) lse->fill_(-INFINITY);
    return {out, lse};
  }
  const Tensor q = rows(query), lens = seq_lens.contiguous();
  const Tensor table = block_table.stride(1) == 1 ? block_table : block_table.contiguous();
  const Tensor start = query_start.has_value() ? query_start->contiguous() : Tensor();
  kvs::Attn4Launch L = {};
  L.q = q.data_ptr(), L.out = out.data_ptr(), L.cache = cache.data_ptr();
  L.table = table.data_ptr<int>(), L.lens = lens.data_ptr<int>();
  if (lse.has_value()) L.lse = lse->data_ptr<float>();
  if (start.defined()) L.start = start.data_ptr<int>();
  L.q_ts = q.stride(0), L.q_hs = q.stride(1), L.o_ts = out.stride(0), L.o_hs = out.stride(1);
  L.block_stride = cache.stride(0), L.head_stride = cache.stride(1);
  L.table_stride = table.stride(0), L.table_cols = int_of("columns", table.size(1));
  L.seqs = int_of("sequences", R), L.tokens = int_of("rows", T);
  L.num_blocks = static_cast<int>(cache.size(0));
  L.q_heads = int_of("query heads", Hq), L.heads = int_of("heads", H);
  L.block_size = static_cast<int>(bs), L.groups = groups, L.causal = causal;
  L.fp16 = query.scalar_type() == at::kHalf;
  L.max_q = static_cast<int>(std::min(max_query_len, T));
  L.scale = static_cast<float>(sc);
  L.clear = !out_in.has_value();
  L.err = g_err[dev.index()];
  const long long bytes = EIGHT ? kvs_attn8_scratch_bytes(&L) : kvs_attn4_scratch_bytes(&L);
  Tensor scratch;  // from the caching allocator: a captured graph has its own
  if (bytes > 0) {
    scratch = at::empty({bytes}, query.options().dtype(at::kByte));
    L.scratch = scratch.data_ptr();
  }
  void* const stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  launched(EIGHT ? kvs_attention_kv8(&L, stream) : kvs_attention_kv4(&L, stream), what);
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception<NoErrorWord>(m, "NoErrorWord");
  m.attr("torch_version") = KVS_TORCH_VERSION;
  m.def("set_error_word", [](int64_t device, int64_t ptr) {
    TORCH_CHECK_VALUE(device >= 0 && device < kMaxDevices, "device index out of range");
    g_err[device] = reinterpret_cast<uint32_t*>(ptr);
  });
  m.def("append_kv", &append_kv);
  m.def("read_kv4", [](const Tensor& cache, const Tensor& slots, py::object dtype,
                       const optional<Tensor>& out) {
    return read_rows<false>(cache, slots, torch::python::detail::py_object_to_dtype(dtype), out);
  });
  m.def("read_kv8", [](const Tensor& cache, const Tensor& slots, py::object dtype,
                       const optional<Tensor>& out) {
    return read_rows<true>(cache, slots, torch::python::detail::py_object_to_dtype(dtype), out);
  });
  m.def("attention_kv4", &attention<false>);
  m.def("attention_kv8", &attention<true>);
}
