// wkf_decode.hpp -- the typed C++ facade over wkf_decode.h, next to wkf_tensor.hpp and in its manner: ranks and element
// types in the types, exceptions for refusals, no state beyond the handles.
#ifndef WKF_DECODE_HPP
#define WKF_DECODE_HPP

#include "wkf_decode.h"
#include "wkf_tensor.hpp"

namespace wkf {

// Weights [k, n] in 4 bits with a scale (and a zero point) for each group of rows and column: wkf_q4_new.  S: the scales' type.
class Q4Weights {
 public:
  template <class S>
  static Q4Weights make(const Device& dev, size_t k, size_t n, size_t group, const std::vector<uint8_t>& codes,
                        const std::vector<typename S::host_type>& scales, const std::vector<uint8_t>& zeros = {}) {
    const size_t groups = group ? k / group + (k % group != 0) : 0;
    if (codes.size() != k * n || scales.size() != groups * n || (!zeros.empty() && zeros.size() != groups * n))
      throw Error(WKF_ERR_INVALID_ARG, "Q4Weights: codes, scales or zeros of another size");
    wkf_q4* h = nullptr;
    check(wkf_q4_new(dev.handle(), k, n, group, codes.data(), S::id, scales.data(), zeros.empty() ? nullptr : zeros.data(), &h));
    return Q4Weights(h);
  }
  wkf_q4* handle() const { return h_.get(); }

 private:
  explicit Q4Weights(wkf_q4* h) : h_(h, wkf_q4_free) {}
  std::shared_ptr<wkf_q4> h_;
};

// Keys and values in 8 bits: wkf_kv_cache_create.
class KvCache {
 public:
  KvCache(const Device& dev, size_t sequences, size_t kv_heads, size_t head_dim, size_t capacity, size_t block = 64) : sequences_(sequences) {
    wkf_kv_cache* h = nullptr;
    check(wkf_kv_cache_create(dev.handle(), sequences, kv_heads, head_dim, capacity, block, &h));
    h_.reset(h, wkf_kv_cache_free);
  }
  std::vector<size_t> lengths() const {
    std::vector<size_t> n(sequences_);
    for (size_t b = 0; b < sequences_; b++) check(wkf_kv_cache_length(h_.get(), b, &n[b]));
    return n;
  }
  void reset(size_t sequence = size_t(-1)) { check(wkf_kv_cache_reset(h_.get(), sequence)); }
  template <int R, class D>
  void append(const Tensor<R, D>& k, const Tensor<R, D>& v, const std::vector<size_t>& counts = {}) {
    static_assert(R == 3 || R == 4, "[sequences, kv_heads, S, head_dim], or one sequence's");
    check(wkf_kv_cache_append(h_.get(), k.handle(), v.handle(), counts_of(counts)));
  }
  template <class D>
  Tensor<5, D> values(size_t first, size_t count) const {
    wkf_tensor* t = nullptr;
    check(wkf_kv_cache_values(h_.get(), D::id, first, count, &t));
    return Tensor<5, D>::adopt(t);
  }
  wkf_kv_cache* handle() const { return h_.get(); }
  const size_t* counts_of(const std::vector<size_t>& counts) const {
    if (counts.empty()) return nullptr;
    if (counts.size() != sequences_) throw Error(WKF_ERR_INVALID_ARG, "one count per sequence is required");
    return counts.data();
  }

 private:
  size_t sequences_;
  std::shared_ptr<wkf_kv_cache> h_;
};

template <int R, class D>
Tensor<R, D> mat_mul_q4(const Tensor<R, D>& x, const Q4Weights& w) {
  wkf_tensor* t = nullptr;
  check(wkf_tensor_mat_mul_q4(x.handle(), w.handle(), &t));
  return Tensor<R, D>::adopt(t);
}

// W, C: the element types of weight and tables (D or F32)
template <int R, class D, class W, class C>
Tensor<R, D> norm_rope(const Tensor<R, D>& x, const Tensor<1, W>& weight, const Tensor<2, C>& cos, const Tensor<2, C>& sin, float eps,
                       const std::vector<size_t>& positions = {}) {
  static_assert(R == 3 || R == 4, "[heads, seq, dim] or [batch, heads, seq, dim]");
  if (!positions.empty() && positions.size() != (R == 4 ? x.shape()[0] : size_t(1)))
    throw Error(WKF_ERR_INVALID_ARG, "norm_rope: one position per batch entry is required");
  wkf_tensor* t = nullptr;
  check(wkf_tensor_norm_rope(x.handle(), weight.handle(), cos.handle(), sin.handle(), eps, positions.empty() ? nullptr : positions.data(), &t));
  return Tensor<R, D>::adopt(t);
}

template <int R, class D>
Tensor<R, D> attend(const Tensor<R, D>& q, const KvCache& cache, float scale, bool causal = true, const std::vector<size_t>& counts = {}) {
  static_assert(R == 3 || R == 4, "[sequences, heads, S, head_dim], or one sequence's");
  wkf_tensor* t = nullptr;
  check(wkf_tensor_attend(q.handle(), cache.handle(), scale, causal ? 1 : 0, cache.counts_of(counts), &t));
  return Tensor<R, D>::adopt(t);
}

template <int R, class D>
Tensor<R, D> zeros(const Device& dev, const std::array<size_t, size_t(R)>& shape) {
  wkf_tensor* t = nullptr;
  check(wkf_tensor_zeros(dev.handle(), D::id, R, shape.data(), &t));
  return Tensor<R, D>::adopt(t);
}

template <int R, class D>
void materialize_into(const Tensor<R, D>& t, const Tensor<R, D>& out) {
  wkf_tensor *from = t.handle(), *to = out.handle();
  check(wkf_tensor_materialize_into(&from, 1, &to));
}

// One of several tensors and where it goes, in the braces of the call below; tensors of any rank and type stand beside each other.
struct Into {
  template <int R, class D>
  Into(const Tensor<R, D>& t, const Tensor<R, D>& out) : from(t.handle()), to(out.handle()) {}
  wkf_tensor *from, *to;
};
// materialize_into({{q, out_q}, {k, out_k}}): one pass over the joint graph, in which sibling norm_ropes are one launch.
inline void materialize_into(std::initializer_list<Into> list) {
  std::vector<wkf_tensor*> from, to;
  for (const Into& i : list) {
    from.push_back(i.from);
    to.push_back(i.to);
  }
  check(wkf_tensor_materialize_into(from.data(), int(list.size()), to.data()));
}

}  // namespace wkf

#endif
