// Host side of the operators of a step with trees of drafted tokens: looks over the arguments, allocates the outputs and launches the
// kernels of libxllm_kernels.so (whose entry points Python hands over, so that there is one place that says which library is loaded).
//
// The small ones of these calls take a few microseconds on the GPU; the same work in Python took 20 to 30.  A call whose arguments are
// not as documented launches nothing and returns None: the caller then says what is wrong with them.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "tree_api.h"

namespace py = pybind11;
using at::Tensor;

namespace {

constexpr int64_t kTreeRows = 256;

decltype(&xl_step_rows) f_step_rows;
decltype(&xl_accept_tree) f_accept;
decltype(&xl_attention_tree_workspace) f_workspace;
decltype(&xl_attention_tree) f_attention;
decltype(&xl_adjust_logits) f_logits;

void bind(const std::unordered_map<std::string, uint64_t>& at) {
  f_step_rows = reinterpret_cast<decltype(f_step_rows)>(at.at("xl_step_rows"));
  f_accept = reinterpret_cast<decltype(f_accept)>(at.at("xl_accept_tree"));
  f_workspace = reinterpret_cast<decltype(f_workspace)>(at.at("xl_attention_tree_workspace"));
  f_attention = reinterpret_cast<decltype(f_attention)>(at.at("xl_attention_tree"));
  f_logits = reinterpret_cast<decltype(f_logits)>(at.at("xl_adjust_logits"));
}

using Opt = std::optional<Tensor>;
const void* ptr(const Opt& t) { return t ? t->const_data_ptr() : nullptr; }

struct Like {
  at::Device dev;
  bool operator()(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> sizes) const {
    return t.scalar_type() == type && t.device() == dev && t.sizes().equals(at::IntArrayRef(sizes)) && t.is_contiguous();
  }
};

void check(int rc, const char* name) {
  if (rc != 0)
    throw std::runtime_error(std::string(name) + " failed with code " + std::to_string(rc) + " (-2: unsupported shape/alignment, -1: launch error)");
}

Tensor ints(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kInt)); }

py::object step_rows(const Tensor& tables, const Tensor& lens, const Tensor& seqs, const Tensor& counts, int64_t n_rows, int64_t block,
                     const Opt& parents, int64_t max_q, int64_t max_blocks) {
  const Like like{tables.device()};
  const auto i32 = at::kInt;
  if (tables.dim() != 2 || tables.scalar_type() != i32 || (tables.stride(1) != 1 && tables.size(1) > 1)) return py::none();
  const int64_t pool = tables.size(0), B = seqs.numel();
  if (!like(lens, i32, {pool}) || !like(seqs, i32, {B}) || !like(counts, i32, {B}) || (parents && !like(*parents, i32, {n_rows})) || n_rows < 0 ||
      n_rows > INT32_MAX || block < 1 || block > INT32_MAX || max_q < 1 || max_q > INT32_MAX || max_blocks < 0 || max_blocks > tables.size(1) ||
      B >= 65535 || (parents && max_q > kTreeRows) || tables.size(1) > INT32_MAX)
    return py::none();
  const c10::cuda::CUDAGuard guard(tables.device());
  const at::AutoDispatchBelowADInplaceOrView fresh;                    // the parts of an allocation are outputs of their own, no views
  const int64_t words = parents ? (max_q + 63) / 64 : 0;
  // one allocation for the small outputs
  const Tensor small = ints(tables, {3 * n_rows + 2 * B + 1}), out = ints(tables, {B, max_blocks});
  Opt tree;
  if (parents) tree = at::empty({n_rows, words}, tables.options().dtype(at::kLong));
  int* at = small.data_ptr<int>();
  check(f_step_rows(tables.const_data_ptr(), lens.const_data_ptr(), seqs.const_data_ptr(), counts.const_data_ptr(), ptr(parents), at, at + n_rows,
                    at + 2 * n_rows, at + 3 * n_rows, at + 3 * n_rows + B + 1, out.data_ptr(), tree ? tree->data_ptr() : nullptr, int(pool),
                    int(tables.size(1)), tables.stride(0), int(B), int(n_rows), int(max_q), int(max_blocks), int(block), int(words),
                    c10::cuda::getCurrentCUDAStream().stream()),
        "xl_step_rows");
  auto part = [&](int64_t from, int64_t n) { return small.as_strided({n}, {1}, from); };
  return py::make_tuple(part(0, n_rows), part(n_rows, n_rows), part(2 * n_rows, n_rows), part(3 * n_rows, B + 1), part(3 * n_rows + B + 1, B), out, tree);
}

py::object tree_attention(Tensor q, const Tensor& k, const Tensor& v, const Tensor& q_cu, const Tensor& kv_lens, const Tensor& tables,
                          const Tensor& token_seq, const Tensor& positions, int64_t B, int64_t max_q, int64_t max_kv, const Tensor& tree, double scale,
                          int64_t window) {
  const Like like{q.device()};
  const auto i32 = at::kInt, type = q.scalar_type();
  if (q.dim() != 3 || (type != at::kFloat && type != at::kBFloat16) || k.dim() != 4 || tree.dim() != 2 || tables.dim() != 2 || B < 0) return py::none();
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), blocks = k.size(0), block = k.size(1), Hkv = k.size(2), W = tree.size(1);
  if (!like(k, type, {blocks, block, Hkv, D}) || !like(v, type, {blocks, block, Hkv, D}) || D < 1 || D > 512 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || block < 1 || block > INT32_MAX || W < 1 ||
      W > kTreeRows / 64 || max_q > kTreeRows || !like(tree, at::kLong, {T, W}) || !like(q_cu, i32, {B + 1}) || !like(kv_lens, i32, {B}) ||
      !like(tables, i32, {B, tables.size(1)}) || !like(token_seq, i32, {T}) || !like(positions, i32, {T}) || T * Hq > INT32_MAX || blocks > INT32_MAX ||
      max_kv > INT32_MAX || window > INT32_MAX || window < INT32_MIN)
    return py::none();
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor out = at::empty({T, Hq * D}, q.options());
  // no tensor-core kernel: for scores that do not grow with the product, nor where the caches lie off 16-byte boundaries
  const auto address = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()); };
  const bool f32 = type == at::kFloat, plain = f32 || !(scale > 0) || (address(k) | address(v)) % 16 != 0;
  int tc = 0;
  const long size = f_workspace(int(T), int(B), int(tables.size(1)), int(block), int(blocks), int(Hq), int(Hkv), int(D), plain, int(max_q), int(max_kv), &tc);
  if (q.stride(2) != 1 || (tc && (q.stride(1) < 1 || q.stride(0) < 1 || q.stride(1) % 8 || q.stride(0) % std::max<int64_t>(8, q.stride(1)) ||
                                  address(q) % 16)))
    q = q.clone(at::MemoryFormat::Contiguous);
  Opt work;
  if (size > 0) work = at::empty({size}, q.options().dtype(at::kByte));
  check(f_attention(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.data_ptr(), q_cu.const_data_ptr(), kv_lens.const_data_ptr(),
                    tables.const_data_ptr(), token_seq.const_data_ptr(), positions.const_data_ptr(), tree.const_data_ptr(), int(T), int(B),
                    int(tables.size(1)), int(block), int(blocks), int(Hq), int(Hkv), int(D), int(W), q.stride(0), q.stride(1), float(scale), int(window),
                    f32, int(max_q), int(max_kv), tc, work ? work->data_ptr() : nullptr, size, c10::cuda::getCurrentCUDAStream().stream()),
        "xl_attention_tree");
  return py::cast(out);
}

py::object adjust_logits(const Tensor& logits, const Tensor& q_cu, const Opt& seqs, const Opt& text, const Opt& lens, const Opt& prompts,
                         const Opt& rep, const Opt& freq, const Opt& pres, const Opt& tokens, const Opt& parents, const Opt& bias_cu,
                         const Opt& bias_ids, const Opt& bias_values, const Opt& words, const Opt& mask_of, int64_t max_q) {
  const Like like{logits.device()};
  const auto i32 = at::kInt, f32 = at::kFloat, type = logits.scalar_type();
  if (logits.dim() != 2 || (type != f32 && type != at::kBFloat16) || q_cu.dim() != 1 || q_cu.numel() < 1) return py::none();
  const int64_t S = logits.size(0), V = logits.size(1), B = q_cu.numel() - 1;
  if (V < 1 || (logits.stride(1) != 1 && V > 1) || (logits.stride(0) < V && S > 1) || S > INT32_MAX || V > (1 << 30) || !like(q_cu, i32, {B + 1}))
    return py::none();
  // what comes in several parts is there as a whole or not at all
  const bool history = text || lens || prompts || rep || freq || pres, biased = bias_cu || bias_ids || bias_values;
  if ((history && !(text && lens && prompts && rep && freq && pres)) || (biased && !(bias_cu && bias_ids && bias_values)) || bool(words) != bool(mask_of))
    return py::none();
  int64_t pool = B;
  if (text) {
    pool = lens->numel();
    if (text->scalar_type() != i32 || text->dim() != 2 || text->size(0) != pool || (text->stride(1) != 1 && text->size(1) > 1) ||
        text->device() != like.dev || text->size(1) > INT32_MAX || !like(*lens, i32, {pool}) || !like(*prompts, i32, {pool}) ||
        !like(*rep, f32, {pool}) || !like(*freq, f32, {pool}) || !like(*pres, f32, {pool}))
      return py::none();
  } else if (tokens) {
    return py::none();
  }
  if ((tokens && !like(*tokens, i32, {S})) || (parents && (!tokens || !like(*parents, i32, {S}))) || (seqs && !like(*seqs, i32, {B}))) return py::none();
  int64_t n_bias = 0;
  if (bias_cu) {
    n_bias = bias_ids->numel();
    if (!text) pool = bias_cu->numel() - 1;
    if (pool < 0 || n_bias > INT32_MAX || !like(*bias_cu, i32, {pool + 1}) || !like(*bias_ids, i32, {n_bias}) || !like(*bias_values, f32, {n_bias}))
      return py::none();
  }
  if (words && (words->scalar_type() != i32 || words->dim() != 2 || (words->stride(1) != 1 && words->size(1) > 1) || words->size(1) * 32 < V ||
                words->device() != like.dev || words->stride(0) > INT32_MAX || words->size(0) > INT32_MAX || !like(*mask_of, i32, {S})))
    return py::none();
  if (max_q < 1 || max_q > INT32_MAX || (tokens && max_q > kTreeRows)) return py::none();
  const c10::cuda::CUDAGuard guard(logits.device());
  check(f_logits(logits.data_ptr(), type == f32, int(S), int(V), logits.stride(0), q_cu.const_data_ptr(), ptr(seqs), int(B), int(pool), int(max_q),
                 ptr(text), text ? text->stride(0) : 0, text ? int(text->size(1)) : 0, ptr(lens), ptr(prompts), ptr(rep), ptr(freq), ptr(pres),
                 ptr(tokens), ptr(parents), ptr(bias_cu), ptr(bias_ids), ptr(bias_values), int(n_bias), ptr(words),
                 words ? int(words->stride(0)) : 0, words ? int(words->size(0)) : 0, ptr(mask_of), c10::cuda::getCurrentCUDAStream().stream()),
        "xl_adjust_logits");
  return py::bool_(true);
}

py::object accept_tree(const Tensor& target, const Tensor& tokens, const Tensor& parents, const Tensor& q_cu, const Tensor& kv_lens,
                       const Tensor& tables, int64_t B, int64_t block, int64_t max_q, int64_t depth, const std::vector<Tensor>& caches) {
  const Like like{target.device()};
  const auto i32 = at::kInt;
  const int64_t T = target.numel();
  if (tables.dim() != 2 || B < 0 || B >= 65536 || block < 1 || max_q > kTreeRows || depth < 0 || depth >= kTreeRows || T > INT32_MAX ||
      !like(target, i32, {T}) || !like(tokens, i32, {T}) || !like(parents, i32, {T}) || !like(q_cu, i32, {B + 1}) || !like(kv_lens, i32, {B}) ||
      !like(tables, i32, {B, tables.size(1)}))
    return py::none();
  std::vector<void*> at;
  std::vector<int> rows, blocks;
  std::vector<std::pair<uintptr_t, uintptr_t>> held;                   // first byte of a cache, the one behind its last
  uintptr_t all = 0;
  held.reserve(caches.size());
  at.reserve(caches.size());
  rows.reserve(caches.size());
  blocks.reserve(caches.size());
  for (const Tensor& c : caches) {
    if (c.dim() < 2 || c.size(1) != block || !c.is_contiguous() || c.device() != like.dev || c.size(0) > INT32_MAX) return py::none();
    if (c.numel() == 0) continue;
    const int64_t row = int64_t(c.nbytes()) / (c.size(0) * block);
    if (row > INT32_MAX) return py::none();
    at.push_back(c.data_ptr());
    rows.push_back(int(row));
    blocks.push_back(int(c.size(0)));
    const auto first = reinterpret_cast<uintptr_t>(c.data_ptr());
    held.emplace_back(first, first + c.nbytes());
    all |= first | uintptr_t(row);
  }
  // no memory twice: it would move twice
  std::sort(held.begin(), held.end());
  for (size_t i = 1; i < held.size(); ++i)
    if (held[i].first < held[i - 1].second) return py::none();
  // the widest unit that divides every cache's rows and address
  const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
  for (int& r : rows) r /= unit;
  const c10::cuda::CUDAGuard guard(target.device());
  const at::AutoDispatchBelowADInplaceOrView fresh;
  // one allocation for the outputs
  const Tensor all_out = ints(target, {B * (2 * depth + 3)});
  int* const o = all_out.data_ptr<int>();
  check(f_accept(target.const_data_ptr(), tokens.const_data_ptr(), parents.const_data_ptr(), q_cu.const_data_ptr(), kv_lens.const_data_ptr(),
                 tables.const_data_ptr(), o, o + 2 * B * (depth + 1), o + B * (depth + 1), int(T), int(B), int(tables.size(1)), int(block), int(depth),
                 at.data(), rows.data(), blocks.data(), int(at.size()), unit, c10::cuda::getCurrentCUDAStream().stream()),
        "xl_accept_tree");
  auto rows_of = [&](int64_t from) { return all_out.as_strided({B, depth + 1}, {depth + 1, 1}, from); };
  return py::make_tuple(rows_of(0), all_out.as_strided({B}, {1}, 2 * B * (depth + 1)), rows_of(B * (depth + 1)));
}

}  // namespace

// what build_ext finds in the file when it decides whether to build again
__attribute__((used)) const char kBuiltFor[] = "built for torch " XL_TORCH_VERSION ";";

PYBIND11_MODULE(_tree_host, m) {
  m.def("bind", &bind);
  m.def("step_rows", &step_rows);
  m.def("tree_attention", &tree_attention);
  m.def("adjust_logits", &adjust_logits);
  m.def("accept_tree", &accept_tree);
}
