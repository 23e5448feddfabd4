// The paged cache's operations of the PyTorch-ROCm extension (paged_append, paged_branch,
// paged_accept, tree_attention) over the C ABI of libcugo_hip.so.  Like the engine's operations
// they check their tensors, allocate outputs and scratch with torch, launch on the current stream
// under the tensors' device and never synchronise.
#include "ext_common.h"

#include <cmath>

namespace cugo_ext {
namespace {

using torch::Tensor;
using Optional = c10::optional<Tensor>;

// The cache's tensors, checked against each other.
struct Paged {
  CugoPagedCache c{};
  const Tensor& k;
  Paged(const Tensor& k_in, const Tensor& v, const Tensor& table, const Tensor& length,
        const Tensor& refs, const Tensor& free)
      : k(k_in) {
    TORCH_CHECK(k.is_cuda(), "the cache's k must be a CUDA tensor");
    TORCH_CHECK(k.dim() == 5 && k.is_contiguous(),
                "the cache's k must be contiguous [layers, pages, kv_heads, page, dh]");
    TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.is_contiguous(),
                "the cache's v must be contiguous, of k's shape and dtype");
    switch (k.scalar_type()) {
      case at::kFloat:
        c.dtype = CUGO_DTYPE_F32;
        break;
      case at::kHalf:
        c.dtype = CUGO_DTYPE_F16;
        break;
      case at::kBFloat16:
        c.dtype = CUGO_DTYPE_BF16;
        break;
      default:
        TORCH_CHECK(false, "the cache must be float32, float16 or bfloat16");
    }
    const int64_t page = k.size(3), dh = k.size(4);
    TORCH_CHECK(dh == 32 || dh == 64 || dh == 128 || dh == 256,
                "the cache's dh must be 32, 64, 128 or 256");
    TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128 || page == 256,
                "the cache's page must be 16, 32, 64, 128 or 256");
    TORCH_CHECK(k.numel() > 0, "the cache has no pages");
    TORCH_CHECK(table.dim() == 2 && table.is_contiguous() && table.scalar_type() == at::kInt &&
                    table.numel() > 0,
                "the cache's table must be a contiguous int32 [rows, width] tensor");
    check_1d(length, at::kLong, "the cache's length");
    check_1d(refs, at::kInt, "the cache's refs");
    check_1d(free, at::kLong, "the cache's free");
    TORCH_CHECK(length.numel() == table.size(0), "the cache's length must have one entry per row");
    TORCH_CHECK(refs.numel() == k.size(1), "the cache's refs must have one entry per page");
    TORCH_CHECK(free.numel() == (k.size(1) + 63) / 64, "the cache's free must have one bit per page");
    for (const Tensor* t : {&v, &table, &length, &refs, &free})
      check_same_device(k, *t, "the cache's k", "its other tensors");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.table = table.data_ptr<int32_t>();
    c.length = length.data_ptr<int64_t>();
    c.refs = refs.data_ptr<int32_t>();
    c.free = reinterpret_cast<uint64_t*>(free.data_ptr<int64_t>());
    c.layers = k.size(0), c.pages = k.size(1), c.kv_heads = k.size(2), c.page = page, c.dh = dh;
    c.rows = table.size(0), c.width = table.size(1);
  }
  void check(const Tensor& t, const char* name) const {
    check_1d(t, at::kLong, name);
    check_same_device(k, t, "the cache", name);
  }
  void check_layer(int64_t layer) const {
    TORCH_CHECK(layer >= 0 && layer < c.layers, "the cache has no layer ", layer);
  }
};

// [n, heads, dh] whose (heads, dh) blocks are contiguous and 16-byte aligned, n's stride free.
Tensor blocks(const Tensor& t) {
  const bool dense = t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2));
  const bool near = t.size(0) <= 1 || (t.stride(0) >= t.size(1) * t.size(2) &&
                                       t.stride(0) * t.element_size() % 16 == 0);
  const bool aligned = (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
  return dense && near && aligned ? t : t.detach().clone(at::MemoryFormat::Contiguous);
}
int64_t block_stride(const Tensor& t) {
  return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0);
}

Tensor paged_append(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& length,
                    const Tensor& refs, const Tensor& free, int64_t layer, const Tensor& k_new,
                    const Tensor& v_new, const Tensor& pos, const Optional& rows, const Optional& out) {
  const Paged p(k, v, table, length, refs, free);
  p.check_layer(layer);
  TORCH_CHECK(k_new.dim() == 3 && k_new.size(1) == p.c.kv_heads && k_new.size(2) == p.c.dh &&
                  v_new.sizes() == k_new.sizes(),
              "k_new and v_new must have shape [n, kv_heads, dh] of the cache");
  TORCH_CHECK(k_new.scalar_type() == k.scalar_type() && v_new.scalar_type() == k.scalar_type(),
              "k_new and v_new must have the cache's dtype");
  check_same_device(k, k_new, "the cache", "k_new");
  check_same_device(k, v_new, "the cache", "v_new");
  p.check(pos, "pos");
  const int64_t n = k_new.size(0);
  TORCH_CHECK(pos.numel() == n, "pos must have one entry per token");
  if (rows.has_value()) {
    p.check(*rows, "rows");
    TORCH_CHECK(rows->numel() == n, "rows must have one entry per token");
  }
  const DeviceGuard guard(k.device());
  const Tensor kn = blocks(k_new), vn = blocks(v_new);
  const auto ok = out_or_new(out, {n}, at::kBool, k, "out");
  check_call(cugo_paged_append_ok(&p.c, layer, kn.data_ptr(), block_stride(kn), vn.data_ptr(),
                                  block_stride(vn), pos.data_ptr<int64_t>(),
                                  rows.has_value() ? rows->data_ptr<int64_t>() : nullptr, n, u8p(ok),
                                  stream()),
             "paged_append");
  return ok;
}

Tensor paged_branch(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& length,
                    const Tensor& refs, const Tensor& free, const Tensor& dst, const Tensor& src,
                    const Tensor& want) {
  const Paged p(k, v, table, length, refs, free);
  p.check(dst, "dst");
  p.check(src, "src");
  p.check(want, "length");
  const int64_t n = dst.numel();
  TORCH_CHECK(src.numel() == n && want.numel() == n, "dst, src and length must have one entry each");
  const DeviceGuard guard(k.device());
  const auto ok = torch::empty({n}, on(k, at::kBool));
  const int64_t bytes = cugo_paged_branch_workspace(&p.c, n);
  const auto scratch = torch::empty({bytes}, on(k, at::kByte));
  check_call(cugo_paged_branch(&p.c, dst.data_ptr<int64_t>(), src.data_ptr<int64_t>(),
                               want.data_ptr<int64_t>(), n, u8p(ok),
                               bytes ? scratch.data_ptr() : nullptr, bytes, stream()),
             "paged_branch");
  return ok;
}

Tensor paged_accept(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& length,
                    const Tensor& refs, const Tensor& free, const Tensor& rows, const Tensor& start,
                    const Tensor& keep) {
  const Paged p(k, v, table, length, refs, free);
  p.check(rows, "rows");
  p.check(start, "start");
  const int64_t n = rows.numel();
  TORCH_CHECK(start.numel() == n, "rows and start must have one entry each");
  TORCH_CHECK(keep.is_cuda() && keep.dim() == 2 && keep.size(0) == n &&
                  keep.scalar_type() == at::kLong,
              "keep must be a CUDA int64 [n, most] tensor");
  TORCH_CHECK(keep.size(1) <= 1 || keep.stride(1) == 1, "keep must have its last dimension contiguous");
  check_same_device(k, keep, "the cache", "keep");
  const DeviceGuard guard(k.device());
  const auto ok = torch::empty({n}, on(k, at::kBool));
  const int64_t bytes = cugo_paged_accept_workspace(&p.c, n);
  const auto scratch = torch::empty({bytes}, on(k, at::kByte));
  check_call(cugo_paged_accept(&p.c, rows.data_ptr<int64_t>(), start.data_ptr<int64_t>(),
                               keep.numel() ? keep.data_ptr<int64_t>() : nullptr, keep.stride(0),
                               keep.size(1), n, u8p(ok), bytes ? scratch.data_ptr() : nullptr,
                               bytes, stream()),
             "paged_accept");
  return ok;
}

Tensor tree_attention(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& length,
                      const Tensor& refs, const Tensor& free, int64_t layer, const Tensor& q_in,
                      const Tensor& prefix, const Optional& mask, const Optional& rows,
                      const Optional& offsets, c10::optional<double> scale, const Optional& out_in) {
  const Paged p(k, v, table, length, refs, free);
  p.check_layer(layer);
  TORCH_CHECK(q_in.dim() == 3 && q_in.size(2) == p.c.dh && q_in.size(1) > 0 &&
                  q_in.size(1) % p.c.kv_heads == 0,
              "q must have shape [tokens, heads, dh], heads a multiple of the cache's kv_heads");
  TORCH_CHECK(q_in.scalar_type() == k.scalar_type(), "q must have the cache's dtype");
  check_same_device(k, q_in, "the cache", "q");
  p.check(prefix, "prefix");
  CugoTreeAttention a{};
  a.cache = &p.c;
  a.layer = layer;
  a.tokens = q_in.size(0), a.heads = q_in.size(1), a.n = prefix.numel();
  if (rows.has_value()) {
    p.check(*rows, "rows");
    TORCH_CHECK(rows->numel() == a.n, "rows must have one entry per sequence");
    a.rows = rows->data_ptr<int64_t>();
  }
  if (offsets.has_value()) {
    p.check(*offsets, "offsets");
    TORCH_CHECK(offsets->numel() == a.n + 1, "offsets must have one entry per sequence and one more");
    a.offsets = offsets->data_ptr<int64_t>();
  } else {
    TORCH_CHECK(a.n > 0 ? a.tokens % a.n == 0 : a.tokens == 0,
                "without offsets every sequence has as many queries");
  }
  if (mask.has_value()) {
    TORCH_CHECK(mask->is_cuda() && mask->is_contiguous() && mask->dim() == 2 &&
                    mask->scalar_type() == at::kLong,
                "mask must be a contiguous CUDA int64 [tokens, words] tensor");
    check_same_device(k, *mask, "the cache", "mask");
    a.mask_rows = mask->size(0), a.words = mask->size(1);
    TORCH_CHECK(a.mask_rows == a.tokens ||
                    (!offsets.has_value() && a.n > 0 && a.mask_rows == a.tokens / a.n),
                "mask must have a row for every query, or without offsets one for each of a sequence");
    // a mask without words (nothing drafted is attended) has no memory, but is no missing mask
    a.mask = reinterpret_cast<const uint64_t*>(a.words && a.mask_rows ? mask->data_ptr<int64_t>()
                                                                      : prefix.data_ptr<int64_t>());
  }
  TORCH_CHECK(!scale.has_value() || (std::isfinite(static_cast<float>(*scale) * 1.4426950408889634f) &&
                                     static_cast<float>(*scale) != 0.f),
              "scale must be finite (times log2(e) too) and not 0");
  a.scale = static_cast<float>(scale.value_or(1.0 / std::sqrt(static_cast<double>(p.c.dh))));
  const DeviceGuard guard(k.device());
  const Tensor q = blocks(q_in);
  const auto out = out_or_new(out_in, {a.tokens, a.heads, p.c.dh}, k.scalar_type(), k, "out");
  if (a.tokens == 0) return out;
  a.q = q.data_ptr();
  a.q_stride = block_stride(q);
  a.prefix = prefix.data_ptr<int64_t>();
  a.out = out.data_ptr();
  const int64_t bytes = cugo_tree_attention_workspace(&a);
  const auto scratch = bytes ? torch::empty({bytes}, on(k, at::kByte)) : Tensor();
  check_call(cugo_tree_attention(&a, bytes ? scratch.data_ptr() : nullptr, bytes, stream()),
             "tree_attention");
  return out;
}

}  // namespace

void bind_paged(pybind11::module_& m) {
  namespace py = pybind11;
  const auto none = py::none();
  m.def("paged_append", &paged_append, "New keys and values into their rows' pages, in place; ok [n]",
        py::arg("k"), py::arg("v"), py::arg("table"), py::arg("length"), py::arg("refs"),
        py::arg("free"), py::arg("layer"), py::arg("k_new"), py::arg("v_new"), py::arg("pos"),
        py::arg("rows") = none, py::arg("out") = none);
  m.def("paged_branch", &paged_branch, "Rows become copies of others, sharing their pages; ok [n]",
        py::arg("k"), py::arg("v"), py::arg("table"), py::arg("length"), py::arg("refs"),
        py::arg("free"), py::arg("dst"), py::arg("src"), py::arg("want"));
  m.def("paged_accept", &paged_accept, "The kept ones of rows' last tokens move together; ok [n]",
        py::arg("k"), py::arg("v"), py::arg("table"), py::arg("length"), py::arg("refs"),
        py::arg("free"), py::arg("rows"), py::arg("start"), py::arg("keep"));
  m.def("tree_attention", &tree_attention, "Drafted tokens' attention over a paged cache",
        py::arg("k"), py::arg("v"), py::arg("table"), py::arg("length"), py::arg("refs"),
        py::arg("free"), py::arg("layer"), py::arg("q"), py::arg("prefix"), py::arg("mask") = none,
        py::arg("rows") = none, py::arg("offsets") = none, py::arg("scale") = none,
        py::arg("out") = none);
}

}  // namespace cugo_ext
