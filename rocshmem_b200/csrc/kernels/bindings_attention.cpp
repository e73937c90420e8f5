// Python bindings of the attention operators.
#include <pybind11/pybind11.h>

#include <stdexcept>
#include <string>

#include "attention_kernels.hpp"

namespace py = pybind11;

namespace rocshmem {
namespace kernels {

namespace {
template <typename T>
T *P(uintptr_t v) { return reinterpret_cast<T *>(v); }
void check(int rc, const char *what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + ": CUDA error " + std::to_string(rc));
}
KvCacheArgs cache_of(const py::tuple &t) {
  return KvCacheArgs{P<void>(t[0].cast<uintptr_t>()), P<void>(t[1].cast<uintptr_t>()), P<float>(t[2].cast<uintptr_t>()),
                     P<float>(t[3].cast<uintptr_t>()), t[4].cast<int>(), t[5].cast<int>(), t[6].cast<int>(),
                     t[7].cast<int>(), t[8].cast<int>()};
}
NormRopeArgs norm_rope_of(const py::tuple &t) {
  NormRopeArgs a{};
  int i = 0;
  a.q = P<void>(t[i++].cast<uintptr_t>());
  a.k = P<void>(t[i++].cast<uintptr_t>());
  a.q_token = t[i++].cast<long long>();
  a.q_head = t[i++].cast<long long>();
  a.k_token = t[i++].cast<long long>();
  a.k_head = t[i++].cast<long long>();
  a.q_weight = P<void>(t[i++].cast<uintptr_t>());
  a.k_weight = P<void>(t[i++].cast<uintptr_t>());
  a.positions = P<void>(t[i++].cast<uintptr_t>());
  a.table = P<float>(t[i++].cast<uintptr_t>());
  a.tokens = t[i++].cast<int>();
  a.q_heads = t[i++].cast<int>();
  a.k_heads = t[i++].cast<int>();
  a.dim = t[i++].cast<int>();
  a.rotary = t[i++].cast<int>();
  a.table_rows = t[i++].cast<int>();
  a.eps = t[i++].cast<float>();
  a.interleaved = t[i++].cast<int>();
  a.type = t[i++].cast<int>();
  a.weight_type = t[i++].cast<int>();
  a.wide_positions = t[i++].cast<int>();
  return a;
}
}  // namespace

void bind_attention(py::module_ &m) {
  m.def("qk_norm_rope", [](const py::tuple &args, uintptr_t q_out, uintptr_t k_out, uintptr_t stream) {
    check(qk_norm_rope(norm_rope_of(args), P<void>(q_out), P<void>(k_out), P<void>(stream)), "qk_norm_rope");
  });
  m.def("qk_norm_rope_workspace", [](int dim) { return qk_norm_rope_workspace(dim); });
  m.def("qk_norm_rope_backward", [](const py::tuple &args, uintptr_t gq, uintptr_t gk, uintptr_t dq, uintptr_t dk,
                                    uintptr_t dqw, uintptr_t dkw, uintptr_t workspace, uintptr_t stream) {
    check(qk_norm_rope_backward(norm_rope_of(args), P<void>(gq), P<void>(gk), P<void>(dq), P<void>(dk), P<void>(dqw),
                                P<void>(dkw), P<float>(workspace), P<void>(stream)), "qk_norm_rope_backward");
  });
  m.def("kv_cache_write", [](const py::tuple &cache, uintptr_t k, uintptr_t v, long long k_token, long long k_head,
                             long long v_token, long long v_head, uintptr_t slots, int wide_slots, int tokens, int type,
                             uintptr_t stream) {
    check(kv_cache_write(cache_of(cache), P<void>(k), P<void>(v), k_token, k_head, v_token, v_head, P<void>(slots),
                         wide_slots, tokens, type, P<void>(stream)), "kv_cache_write");
  });
  m.def("kv_cache_read", [](const py::tuple &cache, uintptr_t k_out, uintptr_t v_out, uintptr_t slots, int wide_slots,
                            int tokens, int type, uintptr_t stream) {
    check(kv_cache_read(cache_of(cache), P<void>(k_out), P<void>(v_out), P<void>(slots), wide_slots, tokens, type,
                        P<void>(stream)), "kv_cache_read");
  });
  m.def("paged_attention_workspace", [](const py::tuple &cache, int batch, int heads) {
    return paged_attention_workspace(cache_of(cache), batch, heads);
  });
  m.def("paged_attention", [](const py::tuple &cache, uintptr_t q, long long q_token, long long q_head, uintptr_t table,
                              long long table_stride, uintptr_t lengths, int batch, int heads, int max_pages, int window,
                              float scale, float softcap, int q_type, int out_type, uintptr_t out, uintptr_t lse,
                              uintptr_t workspace, size_t workspace_bytes, uintptr_t stream) {
    const PagedAttentionArgs a{P<void>(q), q_token, q_head, P<int>(table), table_stride, P<int>(lengths), batch, heads,
                               max_pages, window, scale, softcap, q_type, out_type, P<void>(out), P<float>(lse)};
    check(paged_attention(cache_of(cache), a, P<void>(workspace), workspace_bytes, P<void>(stream)), "paged_attention");
  });
  m.def("attention_join", [](uintptr_t outs, uintptr_t lses, long long out_part, long long lse_part, int parts,
                             long long rows, int dim, int in_type, int out_type, uintptr_t out, uintptr_t lse,
                             uintptr_t stream) {
    check(attention_join(P<void>(outs), P<float>(lses), out_part, lse_part, parts, rows, dim, in_type, out_type,
                         P<void>(out), P<float>(lse), P<void>(stream)), "attention_join");
  });
}

}  // namespace kernels
}  // namespace rocshmem
