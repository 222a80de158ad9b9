// The C entry points of include/wkf_decode.h.
#include "wkf_decode.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "decode.h"
#include "tensor_api.h"

using namespace wkf;

struct wkf_q4 {
  std::shared_ptr<const Q4> w;
};
struct wkf_kv_cache {
  std::shared_ptr<KvCache> c;
};

namespace {

void check(int rc) {
  if (rc != WKF_OK) throw Error(rc, wkf_last_error());
}

BufRef buffer(wkf_device* dev, size_t bytes, bool zero = false) {
  wkf_buffer* b = nullptr;
  check(wkf_buffer_alloc(dev, std::max<size_t>(4, (bytes + 3) & ~size_t(3)), zero ? 1 : 0, &b));
  return BufRef(b);
}

DType dtype_of(int d, const char* who) {
  if (d != WKF_F32 && d != WKF_F16) invalid(std::string(who) + ": unknown dtype");
  return DType(d);
}

// a * b, refused where it does not fit the device's address space
size_t times(size_t a, size_t b, const char* who) {
  size_t r;
  if (__builtin_mul_overflow(a, b, &r) || r > (size_t(1) << 47)) invalid(std::string(who) + ": too large");
  return r;
}

// Settings of launches nobody can ask the time of.
Settings untimed(wkf_device* dev) {
  Settings st = settings_for(dev);
  st.timing = false;
  return st;
}

// The [sequences, heads, S, dim] of a tensor that may lack the first dimension for a cache of one sequence.
void cache_shape(const KvCache& c, const wkf_tensor* t, const char* who, const char* name, size_t* heads, size_t* rows) {
  const std::vector<size_t>& s = t->node->shape;
  const std::string what = std::string(who) + ": " + name;
  if (s.size() != 4 && !(s.size() == 3 && c.seqs == 1)) invalid(what + " must be [sequences, heads, S, head_dim]");
  if (s.size() == 4 && s[0] != c.seqs) invalid(what + " has " + std::to_string(s[0]) + " sequences, the cache " + std::to_string(c.seqs));
  if (s[s.size() - 1] != c.dim) invalid(what + " has heads of " + std::to_string(s[s.size() - 1]) + " elements, the cache of " + std::to_string(c.dim));
  if (t->dev != c.dev) invalid(what + " lives on another device than the cache");
  *heads = s[s.size() - 3];
  *rows = s[s.size() - 2];
  if (*rows > 0x3fffffffull) invalid(what + " has too many rows");
}

std::vector<size_t> counts_of(const KvCache& c, const size_t* counts, size_t rows, const char* who) {
  std::vector<size_t> r(c.seqs, rows);
  if (counts)
    for (size_t b = 0; b < c.seqs; b++) {
      if (counts[b] > rows) invalid(std::string(who) + ": a count is larger than the tensor's rows");
      r[b] = counts[b];
    }
  return r;
}

}  // namespace

extern "C" {

int wkf_tensor_zeros(wkf_device* dev, int dtype, int rank, const size_t* shape, wkf_tensor** out) {
  return guarded([&] {
    need(dev, "wkf_tensor_zeros");
    need(out, "wkf_tensor_zeros");
    if (rank < 0 || (rank > 0 && !shape)) invalid("wkf_tensor_zeros: bad rank / shape");
    const DType dt = dtype_of(dtype, "wkf_tensor_zeros");
    std::vector<size_t> sh(shape, shape + rank);
    size_t n = dtype_size(dt);
    for (size_t d : sh) n = d ? times(n, d, "wkf_tensor_zeros") : 0;
    NodeP t = make(NodeKind::Tensor, dt, sh);
    t->data.device = dev;
    t->data.layout = Layout::contiguous(sh);
    t->data.dtype = dt;
    t->data.buffer = buffer(dev, n, true);
    *out = wrap(dev, t);
  });
}

int wkf_tensor_materialize_into(wkf_tensor* const* ts, int n, wkf_tensor* const* outs) {
  return guarded([&] {
    const char* who = "wkf_tensor_materialize_into";
    need(ts, who);
    need(outs, who);
    if (n <= 0) invalid(std::string(who) + ": no tensors");
    std::vector<NodeP> roots;
    std::vector<TensorData> to;
    for (int i = 0; i < n; i++) {
      need(ts[i], who);
      need(outs[i], who);
      if (ts[i]->dev != ts[0]->dev || outs[i]->dev != ts[0]->dev) invalid(std::string(who) + ": tensors of different devices");
      const Node &t = *ts[i]->node, &o = *outs[i]->node;
      if (o.kind != NodeKind::Tensor || !o.data.layout.is_contiguous()) invalid(std::string(who) + ": an output must be a dense tensor that holds data, not a lazy expression");
      if (t.shape != o.shape || t.dtype != o.dtype) invalid(std::string(who) + ": an output must have its tensor's shape and dtype");
      for (int j = 0; j < i; j++)
        if (to[j].buffer.get() == o.data.buffer.get()) invalid(std::string(who) + ": two outputs are the same tensor");
      roots.push_back(ts[i]->node);
      to.push_back(o.data);
    }
    for (int i = 0; i < n; i++) {
      for (LaunchRecord& r : ts[i]->launches)
        if (r.timer) wkf_timer_destroy(r.timer);
      ts[i]->launches.clear();
    }
    // Row kernels whose workgroups wait for each other need a read-back that can compute the tensor again; there is
    // none here, so rows too long for one workgroup take the kernels without that wait.
    Settings st = settings_for(ts[0]->dev);
    st.row_team = false;
    Resolver(ts[0]->dev, st, &ts[0]->launches).resolve_roots_into(roots, to);
  });
}

int wkf_tensor_device_ptr(const wkf_tensor* t, void** out) {
  return guarded([&] {
    need(t, "wkf_tensor_device_ptr");
    need(out, "wkf_tensor_device_ptr");
    if (t->node->kind != NodeKind::Tensor) invalid("wkf_tensor_device_ptr: the tensor must hold data, not be a lazy expression");
    *out = static_cast<char*>(wkf_buffer_ptr(t->node->data.buffer.get())) + t->node->data.layout.offset * dtype_size(t->node->dtype);
  });
}

int wkf_q4_new(wkf_device* dev, size_t k, size_t n, size_t group, const void* codes, int scale_dtype, const void* scales, const void* zeros,
               wkf_q4** out) {
  return guarded([&] {
    const char* who = "wkf_q4_new";
    need(dev, who);
    need(codes, who);
    need(scales, who);
    need(out, who);
    if (!k || !n) invalid("wkf_q4_new: k and n must not be zero");
    if (k > (size_t(1) << 28) || n > (size_t(1) << 28)) invalid("wkf_q4_new: k and n are at most 2^28");
    if (!group || group % 32) invalid("wkf_q4_new: the group must be a multiple of 32");
    auto w = std::make_shared<Q4>();
    w->dev = dev;
    w->k = k;
    w->n = n;
    w->groups = k / group + (k % group != 0);  // (k + group may pass 64 bits)
    w->given_group = group;
    w->group = std::min(group, (k + 31) / 32 * 32);  // one group: its length does not matter
    w->scale_dtype = dtype_of(scale_dtype, who);
    auto high = [](const void* p, size_t bytes) {
      unsigned char any = 0;
      for (size_t i = 0; i < bytes; i++) any |= static_cast<const unsigned char*>(p)[i];
      return any > 15;
    };
    const size_t kn = times(k, n, who), gn = w->groups * n, es = dtype_size(w->scale_dtype);
    if (high(codes, kn)) invalid("wkf_q4_new: a code is larger than 15");
    if (zeros && high(zeros, gn)) invalid("wkf_q4_new: a zero point is larger than 15");
    const size_t tiles = times(w->tiles_k(), w->tiles_n(), who), padded = times(w->tiles_n() * 16, w->groups, who);
    if (tiles > 0x7fffffffull) invalid("wkf_q4_new: too large");
    // a weight is a scale times a whole number of 0 .. 15 (a NaN fails both comparisons)
    w->fits_f16 = true;
    for (size_t i = 0; i < gn; i++) {
      const float s = w->scale_dtype == DType::F16 ? float(static_cast<const _Float16*>(scales)[i]) : static_cast<const float*>(scales)[i];
      w->fits_f16 &= s == 0.f || (std::fabs(s) >= 0x1p-14f && std::fabs(s) <= 65504.f / 15);
    }
    w->codes = buffer(dev, times(tiles, 1024, who));
    w->scales = buffer(dev, padded * es);
    if (zeros) w->zeros = buffer(dev, padded);
    auto up = [&](const void* p, size_t bytes) {
      TensorData t;
      t.device = dev;
      t.buffer = buffer(dev, bytes);
      check(wkf_buffer_upload(t.buffer.get(), 0, p, bytes));
      return t;
    };
    const TensorData c = up(codes, kn), s = up(scales, gn * es), z = zeros ? up(zeros, gn) : TensorData();
    Resolver(dev, untimed(dev), nullptr).pack_q4(*w, c, s, z);
    *out = new wkf_q4{w};
  });
}

void wkf_q4_free(wkf_q4* w) { delete w; }

int wkf_q4_shape(const wkf_q4* w, size_t* k, size_t* n, size_t* group) {
  return guarded([&] {
    need(w, "wkf_q4_shape");
    if (k) *k = w->w->k;
    if (n) *n = w->w->n;
    if (group) *group = w->w->given_group;
  });
}

int wkf_tensor_mat_mul_q4(const wkf_tensor* x, const wkf_q4* w, wkf_tensor** out) {
  return guarded([&] {
    need(x, "wkf_tensor_mat_mul_q4");
    need(w, "wkf_tensor_mat_mul_q4");
    need(out, "wkf_tensor_mat_mul_q4");
    if (x->dev != w->w->dev) invalid("mat_mul_q4: the tensor and the weights live on different devices");
    std::vector<size_t> shape = x->node->shape;
    if (shape.empty() || shape.back() != w->w->k) invalid("mat_mul_q4: the last dimension must be the weights' " + std::to_string(w->w->k));
    shape.back() = w->w->n;
    NodeP n = make(NodeKind::MatMulQ4, x->node->dtype, shape);
    n->a = x->node;
    auto a = std::make_shared<Q4Args>();
    a->w = w->w;
    n->decode = a;
    *out = wrap(x->dev, n);
  });
}

int wkf_tensor_norm_rope(const wkf_tensor* t, const wkf_tensor* weight, const wkf_tensor* cos, const wkf_tensor* sin, float eps, const size_t* positions,
                         wkf_tensor** out) {
  return guarded([&] {
    const char* who = "wkf_tensor_norm_rope";
    need(t, who);
    need(weight, who);
    need(cos, who);
    need(sin, who);
    need(out, who);
    const std::vector<size_t>& s = t->node->shape;
    if (s.size() != 3 && s.size() != 4) invalid("norm_rope: expects [heads, seq, dim] or [batch, heads, seq, dim]");
    const size_t batch = s.size() == 4 ? s[0] : 1, seq = s[s.size() - 2], dim = s[s.size() - 1];
    if (!dim || dim % 2 || dim > 1024) invalid("norm_rope: the last dimension must be even and at most 1024");
    if (s[s.size() - 3] > 0x3fffffull || seq > 0x3fffffffull || batch > 0x3fffffffull) invalid("norm_rope: too large");
    if (weight->node->shape != std::vector<size_t>{dim}) invalid("norm_rope: the weight must be [dim]");
    const std::vector<size_t>& c = cos->node->shape;
    if (c.size() != 2 || sin->node->shape != c || (c[1] != dim && c[1] * 2 != dim)) invalid("norm_rope: the tables must be [positions, dim / 2] or [positions, dim], both alike");
    if (cos->node->dtype != sin->node->dtype) invalid("norm_rope: the tables differ in dtype");
    for (const wkf_tensor* p : {weight, cos, sin}) {
      if (p->dev != t->dev) invalid("norm_rope: tensors live on different devices");
      if (p->node->dtype != t->node->dtype && p->node->dtype != DType::F32) invalid("norm_rope: weight and tables must have the tensor's dtype or f32");
    }
    if (!(eps >= 0.f) || std::isinf(eps)) invalid("norm_rope: eps must be finite and not negative");
    auto a = std::make_shared<NormRopeArgs>();
    a->eps = eps;
    for (size_t b = 0; b < batch; b++) {
      const size_t p = positions ? positions[b] : 0;
      if (p > c[0] || seq > c[0] - p) invalid("norm_rope: the tables end before position " + std::to_string(p) + " + " + std::to_string(seq));
      if (p > 0xffffffffull - seq) invalid("norm_rope: a position does not fit 32 bits");
      a->positions.push_back(uint32_t(p));
    }
    NodeP n = make(NodeKind::NormRope, t->node->dtype, s);
    n->a = t->node;
    n->more = {weight->node, cos->node, sin->node};
    n->decode = a;
    *out = wrap(t->dev, n);
  });
}

int wkf_kv_cache_create(wkf_device* dev, size_t sequences, size_t kv_heads, size_t head_dim, size_t capacity, size_t block, wkf_kv_cache** out) {
  return guarded([&] {
    const char* who = "wkf_kv_cache_create";
    need(dev, who);
    need(out, who);
    if (!sequences || sequences > kMaxSequences) invalid("kv_cache: 1 to " + std::to_string(kMaxSequences) + " sequences");
    if (!kv_heads || kv_heads > 65535) invalid("kv_cache: 1 to 65535 heads");
    if (!head_dim || head_dim > 256) invalid("kv_cache: heads of 1 to 256 elements");
    if (block != 32 && block != 64 && block != 128) invalid("kv_cache: the block must be 32, 64 or 128 tokens");
    if (!capacity || capacity > (size_t(1) << 30)) invalid("kv_cache: a capacity of 1 to 2^30 tokens");
    auto c = std::make_shared<KvCache>();
    c->dev = dev;
    c->seqs = sequences;
    c->heads = kv_heads;
    c->dim = head_dim;
    c->dp = (head_dim + 63) / 64 * 64;
    c->block = block;
    const size_t whole = std::max<size_t>(block, 64);
    c->cap = (capacity + whole - 1) / whole * whole;
    const size_t rows = 2 * sequences * kv_heads;
    c->codes = buffer(dev, times(times(rows, c->cap, who), c->dp, who));
    c->scales = buffer(dev, times(rows, c->cap / block, who) * 4);
    c->staged = buffer(dev, times(2 * rows, block * head_dim, who) * 4);
    c->capacity = capacity;
    c->len.assign(sequences, 0);
    c->slot.assign(sequences, 0);
    *out = new wkf_kv_cache{c};
  });
}

void wkf_kv_cache_free(wkf_kv_cache* c) { delete c; }

int wkf_kv_cache_length(const wkf_kv_cache* c, size_t sequence, size_t* out) {
  return guarded([&] {
    need(c, "wkf_kv_cache_length");
    need(out, "wkf_kv_cache_length");
    if (sequence >= c->c->seqs) invalid("kv_cache_length: no such sequence");
    std::lock_guard<std::mutex> lock(c->c->mu);
    *out = c->c->len[sequence];
  });
}

int wkf_kv_cache_reset(wkf_kv_cache* c, size_t sequence) {
  return guarded([&] {
    need(c, "wkf_kv_cache_reset");
    if (sequence != size_t(-1) && sequence >= c->c->seqs) invalid("kv_cache_reset: no such sequence");
    std::lock_guard<std::mutex> lock(c->c->mu);
    for (size_t b = 0; b < c->c->seqs; b++)
      if (sequence == size_t(-1) || sequence == b) c->c->len[b] = 0;
    c->c->generation++;
  });
}

int wkf_kv_cache_append(wkf_kv_cache* c, const wkf_tensor* k, const wkf_tensor* v, const size_t* counts) {
  return guarded([&] {
    const char* who = "kv_cache_append";
    need(c, who);
    need(k, who);
    need(v, who);
    size_t heads = 0, rows = 0, vheads = 0, vrows = 0;
    cache_shape(*c->c, k, who, "k", &heads, &rows);
    cache_shape(*c->c, v, who, "v", &vheads, &vrows);
    if (heads != c->c->heads || vheads != heads) invalid("kv_cache_append: k and v must have the cache's heads");
    if (rows != vrows) invalid("kv_cache_append: k and v have different numbers of tokens");
    if (k->node->dtype != v->node->dtype) invalid("kv_cache_append: k and v differ in dtype");
    const std::vector<size_t> n = counts_of(*c->c, counts, rows, who);
    Settings st = untimed(c->c->dev);
    st.row_team = false;  // as in wkf_tensor_materialize_into: nothing here could compute k or v a second time
    Resolver(c->c->dev, st, nullptr).append(*c->c, k->node, v->node, n);
  });
}

int wkf_kv_cache_values(wkf_kv_cache* c, int dtype, size_t first, size_t count, wkf_tensor** out) {
  return guarded([&] {
    need(c, "wkf_kv_cache_values");
    need(out, "wkf_kv_cache_values");
    if (first > c->c->capacity || count > c->c->capacity - first) invalid("kv_cache_values: the tokens reach past the capacity");
    const DType dt = dtype_of(dtype, "kv_cache_values");
    NodeP n = make(NodeKind::CacheValues, dt, {2, c->c->seqs, c->c->heads, count, c->c->dim});
    auto a = std::make_shared<CacheArgs>();
    a->c = c->c;
    a->first = first;
    a->count = count;
    {
      std::lock_guard<std::mutex> lock(c->c->mu);
      a->generation = c->c->generation;
    }
    n->decode = a;
    *out = wrap(c->c->dev, n);
  });
}

int wkf_tensor_attend(const wkf_tensor* q, wkf_kv_cache* c, float scale, int causal, const size_t* counts, wkf_tensor** out) {
  return guarded([&] {
    const char* who = "attend";
    need(q, who);
    need(c, who);
    need(out, who);
    size_t heads = 0, rows = 0;
    cache_shape(*c->c, q, who, "q", &heads, &rows);
    if (!heads || heads % c->c->heads) invalid("attend: the query heads must be a multiple of the cache's");
    if (heads > 65535) invalid("attend: at most 65535 query heads");
    if (heads / c->c->heads * rows > 0x7fffff00ull) invalid("attend: too many rows for a key head");
    if (!(scale >= 0.f) || std::isinf(scale)) invalid("attend: the scale must be finite and not negative");
    const std::vector<size_t> n = counts_of(*c->c, counts, rows, who);
    NodeP t = make(NodeKind::Attend, q->node->dtype, q->node->shape);
    auto a = std::make_shared<CacheArgs>();
    a->c = c->c;
    a->scale = scale;
    a->causal = causal != 0;
    {
      std::lock_guard<std::mutex> lock(c->c->mu);
      a->generation = c->c->generation;
      for (size_t b = 0; b < c->c->seqs; b++) {
        if (n[b] > c->c->len[b]) invalid("attend: sequence " + std::to_string(b) + " has " + std::to_string(c->c->len[b]) + " tokens, fewer than its query rows");
        a->counts.push_back(uint32_t(n[b]));
      }
    }
    t->a = q->node;
    t->decode = a;
    *out = wrap(q->dev, t);
  });
}

}  // extern "C"
