// The decoder operators' launches: which kernel a node becomes and what it is given.  The kernels are in kernels/.
#include "decode.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "graph.h"

namespace wkf {

namespace {
const char* const kPrelude =
#include "kernels/prelude.hip.inc"
    ;
const char* const kKvLayout =
#include "kernels/kv_layout.hip.inc"
    ;
const char* const kKvAppend =
#include "kernels/kv_append.hip.inc"
    ;
const char* const kKvValues =
#include "kernels/kv_values.hip.inc"
    ;
const char* const kKvCodes =
#include "kernels/kv_codes.hip.inc"
    ;
const char* const kAttendRows =
#include "kernels/attend_rows.hip.inc"
    ;
const char* const kAttendPrompt =
#include "kernels/attend_prompt.hip.inc"
    ;
const char* const kNormRope =
#include "kernels/norm_rope.hip.inc"
    ;
const char* const kQ4Pack =
#include "kernels/q4_pack.hip.inc"
    ;
const char* const kQ4Dense =
#include "kernels/q4_dense.hip.inc"
    ;
const char* const kQ4Numbers =
#include "kernels/q4_numbers.hip.inc"
    ;
const char* const kQ4Rows =
#include "kernels/q4_rows.hip.inc"
    ;
const char* const kQ4Tile =
#include "kernels/q4_tile.hip.inc"
    ;
const char* const kQ4MatMul =
#include "kernels/q4_mat_mul.hip.inc"
    ;

char* ptr(const BufRef& b) { return static_cast<char*>(wkf_buffer_ptr(b.get())); }
// "name=value name=value ...": a launch's detail (a stream costs more than the launch's other host work)
std::string detail(std::initializer_list<std::pair<const char*, size_t>> list) {
  std::string s;
  s.reserve(96);
  for (const auto& p : list) s.append(s.empty() ? "" : " ").append(p.first).append("=").append(std::to_string(p.second));
  return s;
}
// the first element of a tensor's layout
char* first(const TensorData& t) { return ptr(t.buffer) + t.layout.offset * dtype_size(t.dtype); }

// texts and numbers after each other
struct Piece {
  const char* text;
  size_t number = 0;
  Piece(const char* t) : text(t) {}
  Piece(size_t n) : text(nullptr), number(n) {}
};
std::string joined(std::initializer_list<Piece> list) {
  std::string s;
  s.reserve(96);
  for (const Piece& p : list) p.text ? s.append(p.text) : s.append(std::to_string(p.number));
  return s;
}

std::string define(const char* name, size_t v) { return std::string("#define ") + name + " " + std::to_string(v) + "\n"; }

// Lengths of up to 8, 64 or 256 sequences travel in an argument block: three kernels, so that the usual few do not carry 2 KB.
size_t room_for(size_t sequences) { return sequences <= 8 ? 8 : sequences <= 64 ? 64 : kMaxSequences; }

// workgroups of `threads` along x: a launch has less than 2^32 threads there
uint32_t grid_dim(size_t v, const char* what, size_t threads = 256) {
  if (v > 0xffffffffull / threads) throw Error(WKF_ERR_UNSUPPORTED, std::string(what) + ": too many workgroups");
  return uint32_t(v);
}

size_t compute_units(wkf_device* dev) {
  wkf_props props;
  if (wkf_device_props(dev, &props) != WKF_OK) throw Error(WKF_ERR_HIP, wkf_last_error());
  return size_t(std::max(1, props.compute_units));
}

std::string kv_defines(const KvCache& c, DType dt, size_t nb) {
  return define("WKF_H", dt == DType::F16) + define("D", c.dim) + define("DP", c.dp) + define("T", c.block) + define("NB", nb);
}
std::string kv_signature(const char* what, const KvCache& c, DType dt, size_t nb) {
  return joined({what, "|gfx950|", dtype_name(dt), "|d", c.dim, "|t", c.block, "|nb", nb});
}
}  // namespace

// The value of `n` with its elements dense in row-major order, or at least its last dimension (`rows` true).
TensorData Resolver::rows_dense(const NodeP& n) {
  TensorData t = resolve(n);
  const size_t R = t.layout.rank();
  if (R && t.layout.shape[R - 1] > 1 && t.layout.strides[R - 1] != 1) return make_contiguous(t);
  return t;
}

// ---- products with 4-bit weights ----------------------------------------------------------------

void Resolver::pack_q4(Q4& w, const TensorData& codes, const TensorData& scales, const TensorData& zeros) {
  const bool z = bool(zeros.buffer), sh = w.scale_dtype == DType::F16;
  const std::string sig = std::string("q4_pack|gfx950|") + dtype_name(w.scale_dtype) + (z ? "|zeros" : "");
  wkf_kernel* k = kernel(sig, [&] { return std::string(kPrelude) + define("WKF_SH", sh) + define("WKF_Z", z) + kQ4Pack; });
  struct {
    const void *codes, *scales, *zeros;
    void *out, *out_scales, *out_zeros;
    uint32_t k, n, groups, tiles_k;
  } a = {ptr(codes.buffer), ptr(scales.buffer), z ? ptr(zeros.buffer) : nullptr, ptr(w.codes), ptr(w.scales), z ? ptr(w.zeros) : nullptr,
         uint32_t(w.k), uint32_t(w.n), uint32_t(w.groups), uint32_t(w.tiles_k())};
  launch("q4_pack", sig, "", k, grid_dim(w.tiles_k() * w.tiles_n(), "q4", 64), 1, 1, 64, a);
}

TensorData Resolver::run_mat_mul_q4(const NodeP& n) {
  const Q4& w = *static_cast<const Q4Args&>(*n->decode).w;
  TensorData x = resolve(n->a);
  if (x.layout.strides != Layout::contiguous_strides(x.layout.shape)) x = make_contiguous(x);
  TensorData out = result_of(n.get());
  const size_t M = x.layout.numel() / w.k, N = w.n, Kp = (w.k + 7) / 8 * 8;
  if (!M) return out;
  if (M > 0xfffffull) throw Error(WKF_ERR_UNSUPPORTED, "mat_mul_q4: more than 2^20 - 1 rows");
  const bool z = bool(w.zeros), h = x.dtype == DType::F16;
  const size_t cus = compute_units(dev_);
  auto tiles_of = [&](size_t mt, size_t columns) { return (M + 16 * mt - 1) / (16 * mt) * ((w.tiles_n() + columns - 1) / columns); };
  // Many f16 rows: where no tiles below cover the product with one round of the chip, the weights are written out once, each
  // rounded to f16, and the product is mat_mul's ([1024,4096]x[4096,11008]: 114 us against 130 in tiles of 4-bit weights;
  // [1024,11008]x[11008,4096], which one round covers: 154 against 104).  Weights that would overflow or lose bits in f16
  // stay in the tiles, which round none, and so does everything where the caller wants exact math.
  if (h && w.fits_f16 && !st_.exact_math && M >= 768 && tiles_of(4, 32) > cus && w.tiles_n() <= 65535) return mat_mul_q4_dense(w, x, out, M);
  // the k = 32 steps of a tile that surely share a group, and the group in units of so many
  const size_t step = w.group % 128 == 0 ? 4 : w.group % 64 == 0 ? 2 : 1, units = w.group / (32 * step);
  int shift = -1;
  for (int i = 0; i < 32; i++)
    if (units == size_t(1) << i) shift = i;
  const std::string kind = joined({dtype_name(x.dtype), "|s", dtype_name(w.scale_dtype), z ? "|zeros" : "", "|step", step, shift < 0 ? "|any" : ""});
  auto defines = [&] { return define("WKF_H", h) + define("WKF_SH", w.scale_dtype == DType::F16) + define("WKF_Z", z) + define("STEP", step) + define("POW2", shift >= 0); };
  const std::string d = detail({{"m", M}, {"n", N}, {"k", w.k}, {"group", w.group}});
  // More than 16 rows share x in the LDS; up to 32 beside few columns do not pay for it (24 rows of [4096,4096]: 10.4 us against 11.3).
  if (M > (w.tiles_n() <= cus ? 32 : 16)) {
    // The smallest tiles of which the chip takes all at once, one a compute unit: larger ones read x less often, smaller ones
    // have K shared by more groups of waves ([4096,4096] f16: 256 rows 16.7 us in 32 x 128, 24.9 in 32 x 64, 26.5 in 64 x 128;
    // 1024 rows 41 in 64 x 256, 51 in 64 x 128; f32 256 rows 43 in 32 x 128, 65 in 32 x 64, 65 in 32 x 256).
    struct Tile {
      size_t mt, nt, nw, kw;
    };
    static constexpr Tile f16_tiles[] = {{2, 1, 4, 4}, {2, 2, 4, 4}, {4, 2, 4, 2}, {4, 2, 8, 1}, {4, 4, 8, 1}}, f32_tiles[] = {{2, 1, 4, 2}, {2, 1, 8, 2}, {2, 2, 8, 1}};
    const Tile *tile = h ? f16_tiles : f32_tiles, *last = h ? std::end(f16_tiles) - 1 : std::end(f32_tiles) - 1;
    while (tile < last && tiles_of(tile->mt, tile->nt * tile->nw) > cus) tile++;
    const size_t mt = tile->mt, nt = tile->nt, nw = tile->nw, kw = tile->kw;
    constexpr size_t depth = 2;
    const void* rows = first(x);
    TensorData planes;
    if (!h || w.k % 8 || reinterpret_cast<uintptr_t>(rows) % 16) {
      const size_t pieces = M * (Kp / 8);
      planes = alloc({size_t(h ? 1 : 3), M, Kp}, DType::F16, false);
      const std::string rsig = joined({"q4_rows|gfx950|", dtype_name(x.dtype)});
      wkf_kernel* rk = kernel(rsig, [&] { return std::string(kPrelude) + define("WKF_H", h) + kQ4Rows; });
      struct {
        const void* x;
        void* out;
        uint32_t m, k, stride, pad;
      } ra = {rows, ptr(planes.buffer), uint32_t(M), uint32_t(w.k), uint32_t(Kp), 0};
      launch("q4_rows", rsig, d, rk, grid_dim((pieces + 255) / 256, "mat_mul_q4"), 1, 1, 256, ra);
      rows = ptr(planes.buffer);
    }
    const std::string sig = joined({"q4_tile|gfx950|", kind.c_str(), "|", mt, "x", nt, "x", nw, "x", kw});
    wkf_kernel* k = kernel(sig, [&] {
      return std::string(kPrelude) + defines() + define("MT", mt) + define("NT", nt) + define("NW", nw) + define("KW", kw) + define("DEPTH", depth) + kQ4Numbers + kQ4Tile;
    });
    struct {
      const void *x, *codes, *scales, *zeros;
      void* y;
      uint32_t m, n, stride, group, groups, tiles_k, shift, tiles_n;
    } a = {rows, ptr(w.codes), ptr(w.scales), z ? ptr(w.zeros) : nullptr, first(out),
           uint32_t(M), uint32_t(N), uint32_t(Kp), uint32_t(w.group), uint32_t(w.groups), uint32_t(w.tiles_k()), uint32_t(std::max(shift, 0)), uint32_t(w.tiles_n())};
    launch("q4_tile", sig, d, k, uint32_t((w.tiles_n() + nw * nt - 1) / (nw * nt)), uint32_t((M + 16 * mt - 1) / (16 * mt)), 1, uint32_t(64 * nw * kw), a);
    return out;
  }
  const size_t mt = M <= 16 ? 1 : 2;
  // eight waves, two tiles each on their way ([1,4096]x[4096,11008] f16: 9.0 us, 10.7 with four waves, 10.0 with sixteen, 10.8 with four tiles)
  constexpr size_t waves = 8, pf = 2;
  const std::string sig = joined({"q4_mat_mul|gfx950|", kind.c_str(), "|w", waves, "|pf", pf, "|mt", mt});
  wkf_kernel* k = kernel(sig, [&] {
    return std::string(kPrelude) + defines() + define("WAVES", waves) + define("PF", pf) + define("MT", mt) + kQ4Numbers + kQ4MatMul;
  });
  struct {
    const void *x, *codes, *scales, *zeros;
    void* y;
    uint32_t m, n, k, group, groups, tiles_k, shift, pad;
  } a = {first(x), ptr(w.codes), ptr(w.scales), z ? ptr(w.zeros) : nullptr, first(out),
         uint32_t(M), uint32_t(N), uint32_t(w.k), uint32_t(w.group), uint32_t(w.groups), uint32_t(w.tiles_k()), uint32_t(std::max(shift, 0)), 0};
  launch("q4_mat_mul", sig, d, k, grid_dim(w.tiles_n(), "mat_mul_q4", 64 * waves), uint32_t((M + 16 * mt - 1) / (16 * mt)), 1, uint32_t(64 * waves), a);
  return out;
}

TensorData Resolver::mat_mul_q4_dense(const Q4& w, const TensorData& x_in, const TensorData& out, size_t M) {
  const size_t N = w.n, Kp = (w.k + 7) / 8 * 8;
  const bool z = bool(w.zeros);
  // rows of x that start on 16 bytes: what mat_mul would otherwise see to by itself
  TensorData x = x_in;
  x.layout.shape = {M, w.k};
  x.layout.strides = {w.k, 1};
  if (Kp != w.k) {
    TensorData padded = alloc({M, Kp}, x.dtype, true), corner = padded;
    corner.layout.shape = {M, w.k};
    copy_map(x, corner);
    x = padded;
  }
  TensorData wt = alloc({N, Kp}, x.dtype, false);
  const std::string sig = joined({"q4_dense|gfx950|s", dtype_name(w.scale_dtype), z ? "|zeros" : ""});
  wkf_kernel* k = kernel(sig, [&] { return std::string(kPrelude) + define("WKF_SH", w.scale_dtype == DType::F16) + define("WKF_Z", z) + kQ4Dense; });
  struct {
    const void *codes, *scales, *zeros;
    void* out;
    uint32_t n, k, stride, group, groups, tiles_k;
  } a = {ptr(w.codes), ptr(w.scales), z ? ptr(w.zeros) : nullptr, ptr(wt.buffer), uint32_t(N), uint32_t(w.k), uint32_t(Kp), uint32_t(w.group), uint32_t(w.groups), uint32_t(w.tiles_k())};
  launch("q4_dense", sig, detail({{"n", N}, {"k", w.k}, {"group", w.group}}), k, uint32_t((w.tiles_k() + 3) / 4), uint32_t(w.tiles_n()), 1, 256, a);
  auto leaf = [&](const TensorData& t) {
    NodeP n = std::make_shared<Node>();
    n->kind = NodeKind::Tensor;
    n->dtype = t.dtype;
    n->shape = t.layout.shape;
    n->data = t;
    return n;
  };
  TensorData b = wt;  // [K, N] as the transpose of the dense [N, K]
  std::swap(b.layout.shape[0], b.layout.shape[1]);
  std::swap(b.layout.strides[0], b.layout.strides[1]);
  NodeP mm = std::make_shared<Node>();
  mm->kind = NodeKind::MatMul;
  mm->dtype = x.dtype;
  mm->shape = {M, N};
  mm->a = leaf(x);
  mm->b = leaf(b);
  TensorData flat = out;
  flat.layout = Layout::contiguous({M, N});
  flat.layout.offset = out.layout.offset;
  mat_mul_out_ = &flat;
  run_matmul(mm);
  return out;
}

// ---- norm and rotation of heads -------------------------------------------------------------------

namespace {
constexpr size_t kMaxMembers = 4;  // tensors of one norm_rope launch

const NormRopeArgs& norm_rope_args(const Node* n) { return static_cast<const NormRopeArgs&>(*n->decode); }

// [batch, heads, seq, dim] of a rank-3 or rank-4 node
size_t nr_dim(const Node* n, size_t i) {
  const std::vector<size_t>& s = n->shape;
  return s.size() == 4 ? s[i] : i == 0 ? 1 : s[i - 1];
}
}  // namespace

namespace {
// whether the value of `n` is computed from that of `from`
bool depends(const NodeP& n, const Node* from, std::set<const Node*>* seen) {
  if (!n || n->kind == NodeKind::Tensor || !seen->insert(n.get()).second) return false;
  if (n.get() == from) return true;
  for (const NodeP& m : n->more)
    if (depends(m, from, seen)) return true;
  return depends(n->a, from, seen) || depends(n->b, from, seen);
}
bool depends(const Node* n, const Node* from) {
  std::set<const Node*> seen;
  return depends(n->a, from, &seen) || depends(n->more[0], from, &seen) || depends(n->more[1], from, &seen) || depends(n->more[2], from, &seen);
}
}  // namespace

void Resolver::join_norm_ropes(const std::vector<NodeP>& roots) {
  std::vector<std::vector<const Node*>> groups;
  std::set<const Node*> seen;
  for (const NodeP& r : roots) {
    if (r->kind != NodeKind::NormRope || !seen.insert(r.get()).second || materialized_.count(r.get())) continue;
    bool placed = false;
    for (auto& g : groups) {
      const Node *o = g[0], *n = r.get();
      const NormRopeArgs &x = norm_rope_args(o), &y = norm_rope_args(n);
      if (g.size() < kMaxMembers && o->dtype == n->dtype && nr_dim(o, 0) == nr_dim(n, 0) && nr_dim(o, 2) == nr_dim(n, 2) && nr_dim(o, 3) == nr_dim(n, 3) &&
          o->more[0]->dtype == n->more[0]->dtype && o->more[1] == n->more[1] && o->more[2] == n->more[2] &&
          memcmp(&x.eps, &y.eps, sizeof(float)) == 0 && x.positions == y.positions &&
          std::none_of(g.begin(), g.end(), [&](const Node* m) { return depends(n, m) || depends(m, n); })) {
        g.push_back(n);
        placed = true;
        break;
      }
    }
    if (!placed) groups.push_back({r.get()});
  }
  for (auto& g : groups) {
    if (g.size() < 2) continue;
    std::vector<TensorData> outs = launch_norm_rope(g);
    for (size_t i = 0; i < g.size(); i++) materialized_[g[i]] = outs[i];
  }
}

TensorData Resolver::run_norm_rope(const NodeP& n) { return launch_norm_rope({n.get()})[0]; }

std::vector<TensorData> Resolver::launch_norm_rope(const std::vector<const Node*>& members) {
  const Node* n0 = members[0];
  const NormRopeArgs& args = norm_rope_args(n0);
  const size_t batch = nr_dim(n0, 0), seq = nr_dim(n0, 2), dim = nr_dim(n0, 3);
  // an input's value with the last `dims` dimensions dense; a leaf's own is not copied
  TensorData kept[2 + 2 * kMaxMembers];
  size_t used = 0;
  auto value = [&](const NodeP& n, size_t dims) {
    const TensorData* t = &n->data;
    TensorData& own = kept[used++];
    if (n->kind != NodeKind::Tensor) {
      own = resolve(n);
      t = &own;
    }
    size_t want = 1;
    for (size_t i = t->layout.rank(), k = 0; i-- && k < dims; k++) {
      if (t->layout.shape[i] > 1 && t->layout.strides[i] != want) {
        own = make_contiguous(*t);
        return const_cast<const TensorData*>(&own);
      }
      want *= t->layout.shape[i];
    }
    return t;
  };
  const TensorData &cos = *value(n0->more[1], 2), &sin = *value(n0->more[2], 2);
  const TensorData *xs[kMaxMembers], *ws[kMaxMembers];
  std::vector<TensorData> outs;
  outs.reserve(members.size());
  size_t heads = 0;
  for (const Node* n : members) {
    xs[outs.size()] = value(n->a, 1);
    ws[outs.size()] = value(n->more[0], 1);
    outs.push_back(result_of(n));
    heads += nr_dim(n, 1);
  }
  if (!batch || !seq || !heads) return outs;
  const size_t nb = room_for(std::min(batch, kMaxSequences)), count = members.size();
  const bool full = cos.layout.shape[1] == dim;
  // the widest pieces of at most 16 bytes that the half is a multiple of, and the lanes that hold a half
  size_t v = n0->dtype == DType::F16 ? 8 : 4, lanes = 1;
  while (dim / 2 % v) v /= 2;
  while (lanes < 64 && lanes * v < dim / 2) lanes *= 2;
  const std::string sig = joined({"norm_rope|gfx950|", dtype_name(n0->dtype), "|w", dtype_name(ws[0]->dtype), "|t", dtype_name(cos.dtype), "|d", dim, full ? "|full" : "", "|nb", nb, "|x", count});
  wkf_kernel* k = kernel(sig, [&] {
    return std::string(kPrelude) + define("WKF_H", n0->dtype == DType::F16) + define("WKF_WH", ws[0]->dtype == DType::F16) + define("WKF_TH", cos.dtype == DType::F16) +
           define("D", dim) + define("FULL", full) + define("V", v) + define("LANES", lanes) + define("NB", nb) + define("MEMBERS", count) + kNormRope;
  });
  const size_t e = dtype_size(n0->dtype);
  for (size_t b0 = 0; b0 < batch; b0 += kMaxSequences) {
    const size_t bn = std::min(batch - b0, kMaxSequences);
    // Member[count], then cos, sin, seq, batch, heads, eps, positions[nb]: kernels/norm_rope.hip.inc
    std::vector<unsigned char> block;
    block.reserve(count * 64 + 64 + nb * 4);
    auto put = [&](const void* p, size_t bytes) { block.insert(block.end(), static_cast<const unsigned char*>(p), static_cast<const unsigned char*>(p) + bytes); };
    for (size_t i = 0; i < count; i++) {
      const Layout& l = xs[i]->layout;
      const size_t r = l.rank(), hn = nr_dim(members[i], 1);
      struct {
        const void *x, *y, *w;
        uint64_t sb, sh, ss, yb;
        uint32_t heads, pad;
      } m = {first(*xs[i]) + (r == 4 ? b0 * l.strides[0] * e : 0), first(outs[i]) + b0 * hn * seq * dim * e, first(*ws[i]),
             r == 4 ? l.strides[0] : 0, l.strides[r - 3], l.strides[r - 2], hn * seq * dim, uint32_t(hn), 0};
      put(&m, sizeof(m));
    }
    struct {
      const void *cos, *sin;
      uint32_t seq, batch, heads;
      float eps;
    } t = {first(cos), first(sin), uint32_t(seq), uint32_t(bn), uint32_t(heads), args.eps};
    put(&t, sizeof(t));
    std::vector<uint32_t> pos(args.positions.begin() + b0, args.positions.begin() + b0 + bn);
    pos.resize(nb);
    put(pos.data(), nb * 4);
    LaunchRecord r;
    r.kind = "norm_rope";
    r.signature = sig;
    r.detail = detail({{"batch", bn}, {"heads", heads}, {"seq", seq}, {"dim", dim}, {"tensors", count}});
    r.block[0] = 256;
    const size_t per = 256 / lanes;
    r.grid[0] = grid_dim((bn * heads * seq + per - 1) / per, "norm_rope");
    record(std::move(r), k, block);
  }
  return outs;
}

// ---- the cache and its attention --------------------------------------------------------------------

namespace {
// the strides of a [sequences, heads, S, dim] tensor, or of one without the first dimension
struct Strides4 {
  uint64_t b, h, s;
  explicit Strides4(const Layout& l) : b(l.rank() == 4 ? l.strides[0] : 0), h(l.strides[l.rank() - 3]), s(l.strides[l.rank() - 2]) {}
};

template <size_t NB>
struct AppendArgs {
  const void* in[2];
  void *codes, *scales, *staged;
  uint64_t sb[2], sh[2], ss[2];
  uint32_t heads, cap, seqs, pad;
  uint32_t len[NB], cnt[NB];
};
template <size_t NB>
struct ValuesArgs {
  void* out;
  const void *codes, *scales;
  uint32_t heads, cap, seqs, first, count, pad;
  uint32_t len[NB];
};
template <size_t NB>
struct AttendArgs {
  const void* q;
  void* out;
  const void *codes, *scales;
  void *part, *stat, *done;
  uint64_t sb, sh, ss;
  uint32_t heads, share, rows, seqs, cap, causal;
  float scale;
  uint32_t span, tiles, walks;
  uint32_t len[NB], cnt[NB], start[NB];
};
template <size_t NB>
struct PromptArgs {
  const void* q;
  void* out;
  const void *codes, *scales;
  uint64_t sb, sh, ss;
  uint32_t heads, share, rows, seqs, cap, causal;
  float scale;
  uint32_t tiles, pairs, pad;
  uint32_t len[NB], cnt[NB];
};

// `f` with the argument block of the cache's size class
template <template <size_t> class A, typename F>
void with_room(size_t nb, F&& f) {
  if (nb == 8) {
    A<8> a = {};
    f(a);
  } else if (nb == 64) {
    A<64> a = {};
    f(a);
  } else {
    A<kMaxSequences> a = {};
    f(a);
  }
}
}  // namespace

void Resolver::append(KvCache& c, const NodeP& kn, const NodeP& vn, const std::vector<size_t>& counts) {
  // what k and v take to compute is launched before the cache is looked at
  std::vector<TensorData> in = resolve_roots({kn, vn});
  for (TensorData& t : in)
    if (t.layout.shape.back() > 1 && t.layout.strides.back() != 1) t = make_contiguous(t);
  std::lock_guard<std::mutex> lock(c.mu);
  size_t blocks = 0, total = 0;
  for (size_t b = 0; b < c.seqs; b++) {
    if (counts[b] > c.capacity - c.len[b])
      invalid("kv_cache_append: sequence " + std::to_string(b) + " would have " + std::to_string(c.len[b] + counts[b]) + " tokens, the cache has room for " + std::to_string(c.capacity));
    total += counts[b];
    if (counts[b]) blocks = std::max(blocks, (c.len[b] + counts[b] - 1) / c.block - c.len[b] / c.block + 1);
  }
  if (!total) return;
  const size_t nb = room_for(c.seqs);
  const std::string sig = kv_signature("kv_append", c, kn->dtype, nb);
  size_t v = kn->dtype == DType::F16 ? 8 : 4;
  while (c.dim % v) v /= 2;
  wkf_kernel* k = kernel(sig, [&] { return std::string(kPrelude) + define("V", v) + kv_defines(c, kn->dtype, nb) + kKvLayout + kKvAppend; });
  with_room<AppendArgs>(nb, [&](auto& a) {
    for (int i = 0; i < 2; i++) {
      const Strides4 st(in[i].layout);
      a.in[i] = first(in[i]);
      a.sb[i] = st.b;
      a.sh[i] = st.h;
      a.ss[i] = st.s;
    }
    a.codes = ptr(c.codes);
    a.scales = ptr(c.scales);
    a.staged = ptr(c.staged);
    a.heads = uint32_t(c.heads);
    a.cap = uint32_t(c.cap);
    a.seqs = uint32_t(c.seqs);
    for (size_t b = 0; b < c.seqs; b++) {
      a.len[b] = c.len[b];
      a.cnt[b] = uint32_t(counts[b]) | uint32_t(c.slot[b]) << 31;
    }
    launch("kv_append", sig, "tokens=" + std::to_string(total), k, grid_dim(blocks, "kv_cache_append"), uint32_t(c.heads), uint32_t(2 * c.seqs), 256, a);
  });
  c.generation++;
  for (size_t b = 0; b < c.seqs; b++) {
    if (!counts[b]) continue;
    const size_t end = c.len[b] + counts[b];
    if ((end - 1) / c.block != c.len[b] / c.block) c.slot[b] ^= 1;  // the block that is open now was staged in the other slot
    c.len[b] = uint32_t(end);
  }
}

TensorData Resolver::run_cache_values(const NodeP& n) {
  const CacheArgs& args = static_cast<const CacheArgs&>(*n->decode);
  KvCache& c = *args.c;
  std::lock_guard<std::mutex> lock(c.mu);
  if (c.generation != args.generation) invalid("kv_cache_values: the cache has been appended to or reset since this tensor was recorded");
  TensorData out = result_of(n.get());
  if (!args.count) return out;
  const size_t nb = room_for(c.seqs);
  const std::string sig = kv_signature("kv_values", c, n->dtype, nb);
  size_t v = n->dtype == DType::F16 ? 8 : 4;
  while (c.dim % v) v /= 2;
  wkf_kernel* k = kernel(sig, [&] { return std::string(kPrelude) + define("V", v) + kv_defines(c, n->dtype, nb) + kKvLayout + kKvValues; });
  with_room<ValuesArgs>(nb, [&](auto& a) {
    a.out = first(out);
    a.codes = ptr(c.codes);
    a.scales = ptr(c.scales);
    a.heads = uint32_t(c.heads);
    a.cap = uint32_t(c.cap);
    a.seqs = uint32_t(c.seqs);
    a.first = uint32_t(args.first);
    a.count = uint32_t(args.count);
    std::copy(c.len.begin(), c.len.end(), a.len);
    const size_t fours = (args.first + args.count + 3) / 4 - args.first / 4, threads = fours * (c.dim / v);
    launch("kv_values", sig, "tokens=" + std::to_string(args.count), k, grid_dim((threads + 255) / 256, "kv_cache_values"), uint32_t(c.heads), uint32_t(2 * c.seqs), 256, a);
  });
  return out;
}

TensorData Resolver::run_attend(const NodeP& n) {
  const CacheArgs& args = static_cast<const CacheArgs&>(*n->decode);
  KvCache& c = *args.c;
  TensorData q = rows_dense(n->a);
  std::lock_guard<std::mutex> lock(c.mu);
  if (c.generation != args.generation) invalid("attend: the cache has been appended to or reset since this tensor was recorded");
  TensorData out = result_of(n.get());
  const size_t R = n->shape.size(), rows = n->shape[R - 2], heads = n->shape[R - 3];
  if (!out.layout.numel()) return out;
  const size_t nb = room_for(c.seqs), share = heads / c.heads, tiles = (share * rows + 15) / 16;
  const size_t cus = compute_units(dev_);
  // Many rows take the kernel that spreads the codes in the LDS for 128 of them; it does not split a cache over workgroups, which
  // the kernel for tiles of 16 rows does.  What counts is how many full tiles of the longest sequence's length all rows come
  // to, each by its own sequence: rows behind a count are no work, and one token over a long cache is one row of a tile that
  // walks all of it alone (2048 new tokens beside 15 single ones over 32768, 32/8 heads of 128 in f16: 36 such tiles, 427 us
  // in tiles of 16 rows and 1408 in tiles of 128; beside 15 over 2000: 516, 275 and 215).  The two meet at about 140 of them in
  // f16 (new tokens up to 4096, 32/8 heads of 128: 512, which are 128 tiles, 90 and 104 us; 640, 160, 108 and 104; 768, 192, 126 and
  // 105), at 175 with heads of 192 (145 and 155; 169 and 156), and at 220 where a tile takes a compute unit alone (f32, heads of
  // 128: 768 tokens 244 and 269, 896, 224, 273 and 268) or the registers do not hold its sums (f16, heads of 256: 1024 tokens,
  // 256, 358 and 326).
  double work = 0;
  size_t furthest = 0;
  for (size_t b = 0; b < c.seqs; b++) {
    if (!args.counts[b]) continue;
    work += double(c.heads * share * args.counts[b]) * c.len[b];
    furthest = std::max<size_t>(furthest, c.len[b]);
  }
  const bool h = n->dtype == DType::F16;
  const double full = double(cus) * (!h ? 0.875 : c.dp <= 128 ? 0.5625 : c.dp <= 192 ? 0.75 : 1.0);
  const size_t big = (share * rows + 127) / 128;
  if (share * rows > 64 && furthest && work >= full * 128 * double(furthest)) {
    const size_t weight_parts = !h ? 3 : st_.exact_math ? 2 : 1;
    const std::string psig = kv_signature("attend_prompt", c, n->dtype, nb) + joined({"|p", weight_parts});
    wkf_kernel* pk = kernel(psig, [&] { return std::string(kPrelude) + define("WEIGHT_PARTS", weight_parts) + kv_defines(c, n->dtype, nb) + kKvLayout + kKvCodes + kAttendPrompt; });
    with_room<PromptArgs>(nb, [&](auto& a) {
      const Strides4 st(q.layout);
      a.q = first(q);
      a.out = first(out);
      a.codes = ptr(c.codes);
      a.scales = ptr(c.scales);
      a.sb = st.b;
      a.sh = st.h;
      a.ss = st.s;
      a.heads = uint32_t(c.heads);
      a.share = uint32_t(share);
      a.rows = uint32_t(rows);
      a.seqs = uint32_t(c.seqs);
      a.cap = uint32_t(c.cap);
      a.causal = args.causal;
      a.scale = args.scale;
      a.tiles = uint32_t(big);
      a.pairs = c.dp <= 128 && h && big * c.heads * c.seqs <= 2 * cus;
      std::copy(c.len.begin(), c.len.end(), a.len);
      std::copy(args.counts.begin(), args.counts.end(), a.cnt);
      launch("attend_prompt", psig, detail({{"sequences", c.seqs}, {"heads", heads}, {"kv_heads", c.heads}, {"rows", rows}, {"dim", c.dim}}), pk, grid_dim(big * c.heads * c.seqs, "attend"), 1, 1, 256, a);
    });
    return out;
  }
  // How many groups of 32 tokens a workgroup takes: so few that there are nearly as many workgroups as the chip holds at once
  // (two a compute unit; large heads leave registers for one), and no more, where a second round would begin (16 sequences of 17000 to 32768
  // tokens, 8 key heads: 149 us, against 174 with 304 workgroups; 8 sequences of up to 3000, 8 heads of 256: 26 us, 33 with
  // 512).  Joining s parts costs about as much as reading s groups, so a few long sequences are split no finer than the square
  // root of twice their groups (one sequence, 8 key heads: 4000 tokens 16.6 us in 32 parts, 11.9 in 8; 16000 tokens 21.4 us in 32
  // parts, 19.3 in 16).  Up to 16 groups stay whole: the join alone takes 3 us.
  // Rows behind a sequence's count see nothing: only the tiles up to it are work.
  size_t total = 0, longest = 0, units = 0;
  std::vector<size_t> live(c.seqs), groups(c.seqs);  // tiles of a key head with rows that see tokens, groups that its rows walk
  for (size_t b = 0; b < c.seqs; b++) {
    live[b] = (share * args.counts[b] + 15) / 16;
    groups[b] = live[b] ? (c.len[b] + 31) / 32 : 0;
    total += c.heads * live[b] * groups[b];
    units += c.heads * live[b];
    longest = std::max(longest, groups[b]);
  }
  constexpr size_t waves = 4, ahead = 2;
  const size_t resident = c.dp <= 128 ? 2 * cus : cus;
  size_t span = longest <= 16 ? longest : std::max((total + resident - 1) / resident, size_t(std::ceil(std::sqrt(2.0 * double(longest)))));
  span = std::max(waves, (span + waves - 1) / waves * waves);
  // Sequences and heads that are more than that by themselves stay whole (64 of 2000 to 4000 tokens, 8 heads: 81 us, 88 in
  // parts), unless some are much longer than the average: half as many again are for those (one of 32000 tokens among 63 of
  // 300: 32 us against 194).  Many times as many keep the chip busy in any case, and their parts would take too much memory.
  const size_t most = std::max(resident, units + (longest * units > 2 * total ? resident / 2 : 0));
  if (units > 32 * resident) span = std::max(span, (longest + waves - 1) / waves * waves);
  auto parts = [&](size_t b) { return std::max<size_t>(1, (groups[b] + span - 1) / span); };
  while (span < longest) {
    size_t workgroups = 0;
    for (size_t b = 0; b < c.seqs; b++) workgroups += c.heads * live[b] * parts(b);
    if (workgroups <= most) break;
    span += (span / 16 + waves) / waves * waves;
  }
  std::vector<uint32_t> start;  // the workgroups of the sequences before each
  size_t walks = 0, dead = 0;
  bool split = false;
  for (size_t b = 0; b < c.seqs; b++) {
    start.push_back(uint32_t(walks));
    walks += c.heads * live[b] * parts(b);
    split |= parts(b) > 1;
    if (live[b] < tiles) dead = c.seqs * c.heads * tiles;
  }
  const uint32_t grid = grid_dim(walks + dead, "attend");
  TensorData part, stat;
  if (split) {
    part = alloc({walks, 16, c.dp}, DType::F32, false);
    stat = alloc({walks, 32}, DType::F32, false);
    if (walks > c.counters) {  // zeros, and every launch leaves zeros
      c.done = alloc({walks}, DType::F32, true).buffer;
      c.counters = walks;
    }
  }
  // A second part of f16 weights costs next to nothing where memory or latency bounds the kernel, with one tile of rows
  // (one token over 1000: 9.2 us and 9.4; 16 sequences of up to 32768: 148 and 149), and more where the products do (512 new
  // tokens after 3584: 87 and 98 us; in tiles of 128, 2048 after 2048: 126 and 169): there it is the caller's choice.
  const size_t weight_parts = !h ? 3 : st_.exact_math || tiles == 1 ? 2 : 1;
  const std::string sig = kv_signature("attend_rows", c, n->dtype, nb) + joined({"|w", waves, "|p", weight_parts});
  wkf_kernel* k = kernel(sig, [&] { return std::string(kPrelude) + define("W", waves) + define("WEIGHT_PARTS", weight_parts) + define("AHEAD", ahead) + kv_defines(c, n->dtype, nb) + kKvLayout + kKvCodes + kAttendRows; });
  const std::string d = detail({{"sequences", c.seqs}, {"heads", heads}, {"kv_heads", c.heads}, {"rows", rows}, {"dim", c.dim}, {"workgroups", walks}});
  with_room<AttendArgs>(nb, [&](auto& a) {
    const Strides4 st(q.layout);
    a.q = first(q);
    a.out = first(out);
    a.codes = ptr(c.codes);
    a.scales = ptr(c.scales);
    a.part = split ? ptr(part.buffer) : nullptr;
    a.stat = split ? ptr(stat.buffer) : nullptr;
    a.done = split ? ptr(c.done) : nullptr;
    a.sb = st.b;
    a.sh = st.h;
    a.ss = st.s;
    a.heads = uint32_t(c.heads);
    a.share = uint32_t(share);
    a.rows = uint32_t(rows);
    a.seqs = uint32_t(c.seqs);
    a.cap = uint32_t(c.cap);
    a.causal = args.causal;
    a.scale = args.scale;
    a.span = uint32_t(span);
    a.tiles = uint32_t(tiles);
    a.walks = uint32_t(walks);
    std::copy(c.len.begin(), c.len.end(), a.len);
    std::copy(args.counts.begin(), args.counts.end(), a.cnt);
    std::copy(start.begin(), start.end(), a.start);
    launch("attend_rows", sig, d, k, grid, 1, 1, uint32_t(64 * waves), a);
  });
  return out;
}

}  // namespace wkf
