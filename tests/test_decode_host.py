"""The decoder operators without a GPU: what the header declares is exported and bound, every refusal, what becomes which
kernel, and the lengths a cache keeps on the host.  On a plan-only device kernels are compiled and nothing is computed."""
import ctypes
import os
import re
import shutil
import subprocess
import sys

import numpy as np
import pytest

from helpers import ROOT

F16, F32 = np.float16, np.float32


def zeros(w, dev, shape, dtype=F32):
    return w.Tensor.new(dev, np.zeros(shape, dtype))


def weights(w, dev, k=64, n=16, group=32, **more):
    g = -(-k // group)
    return w.Q4Weights(dev, np.zeros((k, n), np.uint8), np.ones((g, n), F16), group=group, **more)


def refused(w, match):
    return pytest.raises(w.WkfError, match=match)


def test_header_library_and_binding_agree(wkf):
    text = open(os.path.join(ROOT, "include", "wkf_decode.h")).read()
    declared = set(re.findall(r"\b(wkf_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert declared == set(wkf.DECODE_EXPORTS)
    lib = ctypes.CDLL(wkf.LIB_PATH)
    assert not [n for n in sorted(declared) if not hasattr(lib, n)]


def test_null_arguments_are_refused(wkf, planner):
    lib, h = wkf.load(), ctypes.c_void_p()
    out = ctypes.byref(h)
    t = zeros(wkf, planner, (2, 4, 64))
    cache, q4 = wkf.KvCache(planner, 1, 2, 64, 64), weights(wkf, planner)
    one = (ctypes.c_size_t * 4)(1, 1, 1, 1)
    for rc in (lib.wkf_tensor_zeros(None, 0, 1, one, out), lib.wkf_tensor_zeros(planner._h, 0, 1, one, None), lib.wkf_tensor_zeros(planner._h, 0, 1, None, out),
               lib.wkf_tensor_materialize_into(None, 1, None), lib.wkf_tensor_device_ptr(None, out), lib.wkf_tensor_device_ptr(t._h, None),
               lib.wkf_q4_new(planner._h, 32, 16, 32, None, 0, None, None, out), lib.wkf_q4_shape(None, one, one, one),
               lib.wkf_tensor_mat_mul_q4(None, q4._h, out), lib.wkf_tensor_mat_mul_q4(t._h, None, out), lib.wkf_tensor_mat_mul_q4(t._h, q4._h, None),
               lib.wkf_tensor_norm_rope(t._h, None, None, None, 0.0, None, out), lib.wkf_kv_cache_create(None, 1, 1, 64, 64, 32, out),
               lib.wkf_kv_cache_create(planner._h, 1, 1, 64, 64, 32, None), lib.wkf_kv_cache_length(None, 0, one), lib.wkf_kv_cache_length(cache._h, 0, None),
               lib.wkf_kv_cache_reset(None, 0), lib.wkf_kv_cache_append(cache._h, None, t._h, None), lib.wkf_kv_cache_append(None, t._h, t._h, None),
               lib.wkf_kv_cache_values(None, 0, 0, 1, out), lib.wkf_kv_cache_values(cache._h, 0, 0, 1, None), lib.wkf_tensor_attend(None, cache._h, 1.0, 1, None, out),
               lib.wkf_tensor_attend(t._h, None, 1.0, 1, None, out), lib.wkf_tensor_attend(t._h, cache._h, 1.0, 1, None, None)):
        assert rc == wkf.ERR_INVALID_ARG
    lib.wkf_q4_free(None)
    lib.wkf_kv_cache_free(None)


def test_refusals_of_zeros_and_materialize_into(wkf, planner):
    a, b = zeros(wkf, planner, (3, 4)), zeros(wkf, planner, (3, 4))
    with refused(wkf, "dtype"):
        wkf.Tensor.zeros(planner, (3,), 7)
    with refused(wkf, "too large"):
        wkf.Tensor.zeros(planner, (1 << 40, 1 << 40))
    with refused(wkf, "no tensors"):
        wkf.materialize_into([], [])
    with refused(wkf, "one output per tensor"):
        wkf.materialize_into([a], [])
    with refused(wkf, "lazy expression"):
        wkf.materialize_into([a], [b + 1.0])
    with refused(wkf, "lazy expression"):
        wkf.materialize_into([a.narrow(0, 0, 2)], [b.narrow(0, 0, 2)])
    with refused(wkf, "shape and dtype"):
        wkf.materialize_into([a], [zeros(wkf, planner, (4, 3))])
    with refused(wkf, "shape and dtype"):
        wkf.materialize_into([a], [zeros(wkf, planner, (3, 4), F16)])
    with refused(wkf, "the same tensor"):
        wkf.materialize_into([a + 1.0, a + 2.0], [b, b.clone()])
    other = wkf.Device.planner()
    with refused(wkf, "different devices"):
        wkf.materialize_into([a], [zeros(wkf, other, (3, 4))])
    with refused(wkf, "hold data"):
        (a + 1.0).device_ptr()
    assert a.device_ptr() and not hasattr(a, "__cuda_array_interface__")
    assert wkf.Tensor.zeros(planner, (0, 5)).shape() == (0, 5) and wkf.Tensor.zeros(planner, ()).rank() == 0


def test_refusals_of_weights_in_4_bits(wkf, planner):
    codes, scales = np.zeros((64, 16), np.uint8), np.ones((2, 16), F16)
    for bad, match in [(dict(codes=codes + 16), "0 .. 15"), (dict(codes=codes.astype(int) - 1), "0 .. 15"), (dict(codes=codes.astype(F32)), "whole numbers"),
                       (dict(codes=codes[:0]), "whole numbers"), (dict(codes=codes[0]), "matrix"), (dict(scales=scales[:1]), "scales"),
                       (dict(scales=scales.astype(np.float64)), "scales"), (dict(zeros=np.full((2, 16), 16)), "zeros"), (dict(zeros=np.zeros((1, 16), int)), "zeros"),
                       (dict(group=48), "multiple of 32"), (dict(group=0), "multiple of 32"), (dict(group=-32), "multiple of 32")]:
        with refused(wkf, match):
            wkf.Q4Weights(planner, **{"codes": codes, "scales": scales, "group": 32, **bad})
    lib, h = wkf.load(), ctypes.c_void_p()
    wrong = codes + 16
    p = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    for args in ((0, 16, 32, p(codes), 1, p(scales), None), (64, 0, 32, p(codes), 1, p(scales), None), (64, 16, 33, p(codes), 1, p(scales), None),
                 (64, 16, 32, p(wrong), 1, p(scales), None), (64, 16, 32, p(codes), 1, p(scales), p(wrong)), (64, 16, 32, p(codes), 2, p(scales), None),
                 (1 << 40, 1 << 40, 32, p(codes), 1, p(scales), None)):
        assert lib.wkf_q4_new(planner._h, *args, ctypes.byref(h)) == wkf.ERR_INVALID_ARG
    w = weights(wkf, planner)
    with refused(wkf, "last dimension"):
        zeros(wkf, planner, (3, 63)).mat_mul_q4(w)
    with refused(wkf, "last dimension"):
        zeros(wkf, planner, ()).mat_mul_q4(w)
    with refused(wkf, "different devices"):
        zeros(wkf, wkf.Device.planner(), (3, 64)).mat_mul_q4(w)
    with refused(wkf, "more than 2.20 - 1 rows"):
        zeros(wkf, planner, (1, 64), F16).reshape([64]).broadcast(((1 << 20), 64)).mat_mul_q4(w).materialize()
    y = zeros(wkf, planner, (2, 3, 64), F16).mat_mul_q4(w)
    assert y.shape() == (2, 3, 16) and y.datatype() == wkf.F16
    assert zeros(wkf, planner, (64,)).mat_mul_q4(w).shape() == (16,)


def test_a_group_of_any_size_has_scales_and_zeros(wkf, planner):
    """k rounded up to groups is one group, however large: its zero points are looked at."""
    lib, h = wkf.load(), ctypes.c_void_p()
    codes, scales, zeros = np.zeros((64, 16), np.uint8), np.ones((1, 16), F16), np.full((1, 16), 16, np.uint8)
    p = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    for group in (64, 1 << 63, (1 << 64) - 32):
        assert lib.wkf_q4_new(planner._h, 64, 16, group, p(codes), 1, p(scales), p(zeros), ctypes.byref(h)) == wkf.ERR_INVALID_ARG


def test_the_shape_of_weights_is_what_they_were_made_with(wkf, planner):
    """A group larger than the matrix too, whose length decides nothing."""
    lib = wkf.load()
    for k, n, group in ((64, 16, 32), (64, 16, 4096), (40, 3, 64), (1000, 100, 1024), (33, 1, 1 << 40)):
        w, got = weights(wkf, planner, k, n, group), [ctypes.c_size_t() for _ in range(3)]
        wkf._check(lib.wkf_q4_shape(w._h, *[ctypes.byref(v) for v in got]))
        assert tuple(v.value for v in got) == (k, n, group)


def test_refusals_of_norm_rope(wkf, planner):
    t, g, c = zeros(wkf, planner, (2, 3, 5, 8), F16), zeros(wkf, planner, (8,), F16), zeros(wkf, planner, (9, 4))
    ok = dict(weight=g, cos=c, sin=c, eps=1e-5)
    for bad, match in [(dict(weight=zeros(wkf, planner, (4,), F16)), "weight"), (dict(cos=zeros(wkf, planner, (9, 3))), "tables"), (dict(sin=zeros(wkf, planner, (8, 4))), "tables"),
                       (dict(cos=zeros(wkf, planner, (9, 4), F16)), "differ in dtype"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
                       (dict(positions=[0]), "one position"), (dict(positions=[0, 5]), "tables end"), (dict(positions=[10, 0]), "tables end"),
                       (dict(weight=zeros(wkf, wkf.Device.planner(), (8,), F16)), "different devices")]:
        with refused(wkf, match):
            t.norm_rope(**{**ok, **bad})
    with refused(wkf, "expects"):
        zeros(wkf, planner, (5, 8), F16).norm_rope(**ok)
    with refused(wkf, "even"):
        zeros(wkf, planner, (2, 5, 7)).norm_rope(**ok)
    with refused(wkf, "even"):
        zeros(wkf, planner, (1, 1, 1026)).norm_rope(**ok)
    with refused(wkf, "dtype or f32"):
        zeros(wkf, planner, (2, 5, 8)).norm_rope(**ok)
    assert t.norm_rope(**ok, positions=[4, 0]).shape() == (2, 3, 5, 8)


def test_refusals_of_the_cache_and_its_attention(wkf, planner):
    for bad, match in [(dict(sequences=257), "sequences"), (dict(kv_heads=65536), "heads"), (dict(head_dim=257), "elements"), (dict(block=48), "block"), (dict(block=256), "block"),
                       (dict(capacity=(1 << 30) + 1), "capacity"), (dict(sequences=0), "positive"), (dict(head_dim=-1), "positive"),
                       (dict(sequences=256, kv_heads=65535, head_dim=256, capacity=1 << 30), "too large")]:
        with refused(wkf, match):
            wkf.KvCache(planner, **{"sequences": 2, "kv_heads": 2, "head_dim": 64, "capacity": 40, "block": 32, **bad})
    lib, h = wkf.load(), ctypes.c_void_p()
    assert lib.wkf_kv_cache_create(planner._h, 0, 2, 64, 40, 32, ctypes.byref(h)) == wkf.ERR_INVALID_ARG
    cache = wkf.KvCache(planner, 2, 2, 64, 40, 32)
    k = zeros(wkf, planner, (2, 2, 30, 64))
    for args, match in [((zeros(wkf, planner, (2, 30, 64)), k), "sequences"), ((zeros(wkf, planner, (3, 2, 30, 64)), k), "sequences"), ((k, zeros(wkf, planner, (2, 4, 30, 64))), "heads"),
                        ((k, zeros(wkf, planner, (2, 2, 29, 64))), "different numbers"), ((k, zeros(wkf, planner, (2, 2, 30, 32))), "elements"),
                        ((k, zeros(wkf, planner, (2, 2, 30, 64), F16)), "dtype"), ((k, k, [30, 31]), "count"), ((k, k, [30]), "count per sequence"), ((k, k, [-1, 3]), "count per sequence"),
                        ((k, zeros(wkf, wkf.Device.planner(), (2, 2, 30, 64))), "another device")]:
        with refused(wkf, match):
            cache.append(*args)
    assert cache.lengths() == [0, 0]
    cache.append(k, k, [30, 7])
    with refused(wkf, "room for 40"):
        cache.append(k, k, [0, 30]) or cache.append(k, k, [11, 0])
    assert cache.lengths() == [30, 37]  # a refused append adds nothing, to no sequence
    with refused(wkf, "room for 40"):
        cache.append(k, k, [1, 4])
    assert cache.lengths() == [30, 37]
    q = zeros(wkf, planner, (2, 4, 31, 64), F16)
    for t, more, match in [(q, {}, "fewer than"), (q, dict(counts=[32, 1]), "count"), (zeros(wkf, planner, (2, 3, 1, 64)), {}, "multiple"), (zeros(wkf, planner, (2, 0, 1, 64)), {}, "multiple"),
                           (zeros(wkf, planner, (2, 4, 1, 65)), {}, "elements"), (zeros(wkf, planner, (4, 1, 64)), {}, "sequences"), (q, dict(counts=[1, 1], scale=-1.0), "scale"),
                           (q, dict(counts=[1, 1], scale=float("nan")), "scale"), (q, dict(counts=[1, 1], scale=float("inf")), "scale"),
                           (zeros(wkf, wkf.Device.planner(), (2, 4, 1, 64)), {}, "another device")]:
        with refused(wkf, match):
            t.attend(cache, **more)
    for args in ((0, 41), (40, 1), (41, 0)):
        with refused(wkf, "capacity"):
            cache.values(*args)
    with refused(wkf, "too many rows"):
        zeros(wkf, planner, (2, 8, 64)).broadcast((2, 8, (1 << 30) - 1, 64)).attend(cache, counts=[1, 1])
    with pytest.raises(TypeError):
        zeros(wkf, planner, (2, 4, 1, 64)).attend(cache, counts=[1.5, 1])
    for counts in ([np.int64(1), np.int32(1)], (1, 0)):  # whole numbers of any kind
        assert zeros(wkf, planner, (2, 4, 1, 64)).attend(cache, counts=counts).shape() == (2, 4, 1, 64)
    with refused(wkf, "dtype"):
        cache.values(0, 1, 5)
    with refused(wkf, "no such sequence"):
        cache.reset(2)
    assert lib.wkf_kv_cache_reset(cache._h, 2) == wkf.ERR_INVALID_ARG and lib.wkf_kv_cache_length(cache._h, 2, ctypes.byref(ctypes.c_size_t())) == wkf.ERR_INVALID_ARG
    one = wkf.KvCache(planner, 1, 2, 64, 40, 32)
    one.append(zeros(wkf, planner, (2, 3, 64)), zeros(wkf, planner, (2, 3, 64)))
    assert zeros(wkf, planner, (4, 2, 64)).attend(one).shape() == (4, 2, 64) and one.lengths() == [3]


def test_a_node_stands_for_the_cache_it_was_recorded_with(wkf, planner):
    cache = wkf.KvCache(planner, 1, 1, 64, 40, 32)
    k = zeros(wkf, planner, (1, 1, 4, 64))
    cache.append(k, k)
    early = [zeros(wkf, planner, (1, 1, 1, 64)).attend(cache), cache.values()]
    for t in early:
        t.materialize()
    cache.append(k, k, [0])  # nothing is appended: still the same cache
    for t in early:
        t.materialize()
    cache.append(k, k)
    for t in early:
        with refused(wkf, "appended to or reset"):
            t.materialize()
    out = wkf.Tensor.zeros(planner, (1, 1, 1, 64))
    with refused(wkf, "appended to or reset"):
        wkf.materialize_into([early[0] * 2.0], [out])


def test_handles_may_go_before_what_was_recorded_with_them(wkf, planner):
    w, cache = weights(wkf, planner), wkf.KvCache(planner, 1, 1, 64, 40, 32)
    k = zeros(wkf, planner, (1, 1, 4, 64))
    cache.append(k, k)
    y, o = zeros(wkf, planner, (3, 64)).mat_mul_q4(w), zeros(wkf, planner, (1, 2, 1, 64)).attend(cache)
    del w, cache
    y.materialize()
    o.materialize()


def test_a_device_may_go_before_its_cache_and_weights(wkf):
    dev = wkf.Device.planner()
    w, cache = weights(wkf, dev), wkf.KvCache(dev, 1, 1, 64, 40, 32)
    dev.close()
    del w, cache


def test_what_becomes_which_kernel(wkf, planner):
    x = zeros(wkf, planner, (3, 64), F16)
    y = ((x * 2.0).mat_mul_q4(weights(wkf, planner)) + 1.0).exp()
    y.materialize()
    kinds = [k.kind for k in y.kernels()]
    assert kinds[0] == "map" and kinds[-1] == "map" and "q4_mat_mul" in kinds[1:-1]
    qk = zeros(wkf, planner, (2, 5, 6, 64))
    g, c, d = zeros(wkf, planner, (64,)), zeros(wkf, planner, (9, 32)), zeros(wkf, planner, (9, 32))
    q, k = qk.narrow(2, 0, 4).transpose(1, 2), qk.narrow(2, 4, 2).transpose(1, 2)
    outs = [wkf.Tensor.zeros(planner, (2, 4, 5, 64)), wkf.Tensor.zeros(planner, (2, 2, 5, 64))]

    def kinds_of(a, b):
        wkf.materialize_into([a, b], outs)
        return [n.kind for n in a.kernels()]

    assert kinds_of(q.norm_rope(g, c, c, 1e-5, [1, 2]), k.norm_rope(g, c, c, 1e-5, [1, 2])) == ["norm_rope"]
    # other positions, tables or eps: a launch each
    assert kinds_of(q.norm_rope(g, c, c, 1e-5, [1, 2]), k.norm_rope(g, c, c, 1e-5, [1, 3])) == ["norm_rope"] * 2
    assert kinds_of(q.norm_rope(g, c, c, 1e-5), k.norm_rope(g, d, c, 1e-5)) == ["norm_rope"] * 2
    assert kinds_of(q.norm_rope(g, c, c, 1e-5), k.norm_rope(g, c, c, 1e-6)) == ["norm_rope"] * 2
    # a value that is not an operator's own is computed and copied
    assert kinds_of(q.norm_rope(g, c, c, 1e-5) * 2.0, k.norm_rope(g, c, c, 1e-5)).count("norm_rope") == 2
    dot = q.norm_rope(g, c, c, 1e-5).graphvis()
    assert "norm_rope ([2, 4, 5, 64] f32)" in dot and dot.count("->") >= 4


@pytest.mark.parametrize("reference", [False, True])
def test_a_product_with_written_out_weights_is_left_where_it_is_wanted(wkf, reference):
    """Also where a copy of x has the product's shape: a square matrix, and x that starts behind its buffer's first element."""
    dev = wkf.Device.planner()
    if reference:
        dev.set_fusion(wkf.FUSION_REFERENCE)
    n, m = 6656, 1300
    w = weights(wkf, dev, n, n, 128)
    flat = zeros(wkf, dev, (m * n + 8,), F16)
    for start in (0, 8):
        x = flat.narrow(0, start, m * n).reshape([m, n]) if start else zeros(wkf, dev, (m, n), F16)
        y = x.mat_mul_q4(w)
        wkf.materialize_into([y], [wkf.Tensor.zeros(dev, (m, n), wkf.F16)])
        kinds = [k.kind for k in y.kernels()]
        assert kinds[-1] == "gemm" and kinds.count("q4_dense") == 1, kinds
    dev.close()


def test_written_out_weights_are_f16_only(wkf, planner):
    """Rows of f32 never take them, and the kernel's text has no variant for them."""
    codes = np.zeros((64, 16 * 1024), np.uint8)
    w = wkf.Q4Weights(planner, codes, np.ones((1, 16 * 1024), F16), group=64)
    y, z = zeros(wkf, planner, (1100, 64), F16).mat_mul_q4(w), zeros(wkf, planner, (1100, 64), F32).mat_mul_q4(w)
    y.materialize()
    z.materialize()
    written = [k for k in y.kernels() if k.kind == "q4_dense"]
    assert len(written) == 1 and "WKF_H" not in wkf.kernel_source(written[0].signature)
    assert not [k for k in z.kernels() if k.kind == "q4_dense"]


def test_rows_behind_a_count_are_no_work(wkf, planner):
    """A chunk of a prompt beside single tokens over long caches: the kernel that splits the caches, and as many workgroups
    for that as for the same rows without the empty ones."""
    cache = wkf.KvCache(planner, 4, 8, 64, 8192, 64)
    k = zeros(wkf, planner, (4, 8, 8192, 64), F16)
    cache.append(k, k)

    def launched(rows, counts):
        t = zeros(wkf, planner, (4, 32, rows, 64), F16).attend(cache, counts=counts)
        t.materialize()
        (launch,) = t.kernels()
        return launch.kind, dict(p.split("=") for p in launch.detail.split())

    kind, mixed = launched(256, [256, 1, 1, 1])
    assert kind == "attend_rows" and 512 <= int(mixed["workgroups"]) <= 640
    alone, behind = launched(2, [2, 1, 0, 1]), launched(15, [2, 1, 0, 1])
    assert alone[0] == behind[0] == "attend_rows" and alone[1]["workgroups"] == behind[1]["workgroups"]
    assert launched(1024, [1024] * 4)[0] == "attend_prompt"


def test_extern_block_of_the_guide_matches_the_header():
    """The integration guide declares every function of wkf_decode.h with as many arguments."""
    text = re.sub(r"/\*.*?\*/", " ", open(os.path.join(ROOT, "include", "wkf_decode.h")).read(), flags=re.S)
    c = {m.group(1): m.group(2).count(",") + 1 for m in re.finditer(r"(?:int|void)\s+(wkf_\w+)\s*\(([^;{]*?)\)\s*;", text)}
    guide = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    block = guide[guide.index("// src/ffi_decode.rs"):]
    block = block[:block.index("```")]
    rust = {m.group(1): len([p for p in m.group(2).split(",") if p.strip()]) for m in re.finditer(r"pub fn (wkf_\w+)\s*\(([^)]*)\)", block)}
    assert rust == c


KERNELS = r"""
import sys
import numpy as np
sys.path.insert(0, TESTS)
from helpers import load_package
w = load_package()
dev = w.Device.planner()
T, H, F = w.Tensor, np.float16, np.float32
seen, calls = set(), 0
def done(t):  # a quarter of them each process
    global calls
    calls += 1
    if calls % 4 == int(sys.argv[1]):
        t.materialize()
        seen.update(k.signature for k in t.kernels())
for k, n, ms in ((136, 200, (1, 24, 33)), (160, 2000, (300, 600, 1100)), (130, 7000, (600,)), (64, 11008, (800,))):
    for group in (32, 64, 128):
        for zeros in (None, np.zeros((-(-k // group), n), np.uint8)):
            q4 = w.Q4Weights(dev, np.zeros((k, n), np.uint8), np.ones((-(-k // group), n), H), zeros, group)
            for m in ms:
                for dt in (H, F):
                    done(T.new(dev, np.zeros((m, k), dt)).mat_mul_q4(q4))
for dim in (20, 64, 128, 192, 255, 256):
    for dt in (H, F):
        cache = w.KvCache(dev, 1, 256, dim, 192, 128)
        t = T.new(dev, np.zeros((1, 256, 150, dim), dt))
        cache.append(t, t)
        for q in (t, t.narrow(2, 0, 3), t.narrow(2, 0, 20)):
            done(q.attend(cache))
        done(cache.values(0, 150, w.F16 if dt == H else w.F32))
for dim in (6, 128, 1024):
    for dt in (H, F):
        c = T.new(dev, np.zeros((9, dim), F))
        done(T.new(dev, np.zeros((2, 5, dim), dt)).norm_rope(T.new(dev, np.zeros(dim, dt)), c, c, 1e-5))
print("\n".join(sorted(seen)))
"""


def test_decoder_kernels_use_no_scratch_memory(tmp_path):
    """The compiler's own record of every kernel of these operators: no private segment and no spilled vector register, but for
    two that do not fit: tiles of 128 rows with heads above 192 elements, and the larger tiles of a 4-bit product of f16 rows with
    scales for 32 or 64 rows."""
    from test_host_abi import _code_object_kernels

    def entry(signature):
        h = 1469598103934665603
        for c in signature.encode():
            h = (h ^ c) * 1099511628211 & (1 << 64) - 1
        return f"wkf_{signature.split('|')[0]}_{(h ^ h >> 32) & 0xffffffff:08x}"

    def known(signature):
        dim = re.search(r"^attend_prompt\|.*\|d(\d+)\|", signature)
        return bool(dim and int(dim.group(1)) > 192 or re.search(r"^q4_tile\|gfx950\|f16\|.*\|step[12]\|.*(4x4x8x1|2x2x4x4)$", signature))

    run = [sys.executable, "-c", f"TESTS = {os.path.join(ROOT, 'tests')!r}\n" + KERNELS]
    parts = [subprocess.Popen(run + [str(i)], stdout=subprocess.PIPE, text=True, env=dict(os.environ, WKF_CACHE_DIR=str(tmp_path))) for i in range(4)]
    out = "".join(p.communicate(timeout=900)[0] for p in parts)
    assert not any(p.returncode for p in parts)
    names = {entry(s): s for s in out.split("\n") if s}
    spilled, checked = [], set()
    for path in tmp_path.glob("*.hsaco"):
        for k in _code_object_kernels(path):
            name = k[".name"]
            if not re.match(r"wkf_(q4_|attend_|kv_|norm_rope)", name):
                continue
            checked.add(name.rsplit("_", 1)[0])
            if (k[".private_segment_fixed_size"] or k[".vgpr_spill_count"] or k[".uses_dynamic_stack"]) and not known(names.get(name, "")):
                spilled.append((names.get(name, name), k[".private_segment_fixed_size"], k[".vgpr_spill_count"]))
            assert k[".vgpr_count"] <= 512
    assert not spilled, spilled
    assert checked == {"wkf_" + k for k in ("q4_pack", "q4_rows", "q4_tile", "q4_mat_mul", "q4_dense", "attend_rows", "attend_prompt", "kv_append", "kv_values", "norm_rope")}, checked


FACADE = r"""
    #include <cstdio>
    #include <wkf_decode.hpp>
    using namespace wkf;
    template <class F>
    static int refused(F f) {
      try { f(); } catch (const Error& e) { return e.code; }
      return 0;
    }
    int main() {
      auto dev = Device::planner();
      std::vector<Half> scales(2 * 128, Half::from_float(0.5f));
      auto w = Q4Weights::make<F16>(dev, 64, 128, 32, std::vector<uint8_t>(64 * 128, 3), scales);
      auto y = mat_mul_q4(zeros<2, F16>(dev, {3, 64}), w);
      KvCache cache(dev, 1, 2, 64, 100, 32);
      Tensor<1, F32> g(dev, {64}, std::vector<float>(64, 1.0f));
      auto table = zeros<2, F32>(dev, {9, 32});
      auto k = norm_rope(zeros<3, F16>(dev, {2, 3, 64}), g, table, table, 1e-5f, {6});
      cache.append(k, k);
      cache.append(k, k, {2});
      auto q = norm_rope(zeros<4, F16>(dev, {1, 4, 3, 64}), g, table, table, 1e-5f);
      auto o = attend(q, cache, 0.125f);
      auto out = zeros<4, F16>(dev, {1, 4, 3, 64});
      materialize_into(o, out);
      const bool fine = y.shape() == std::array<size_t, 2>{3, 128} && cache.lengths() == std::vector<size_t>{5} && cache.values<F32>(0, 5).shape()[3] == 5 &&
          refused([&] { cache.append(k, k, {1, 1}); }) == WKF_ERR_INVALID_ARG && refused([&] { norm_rope(k, g, table, table, 1e-5f, {7}); }) == WKF_ERR_INVALID_ARG &&
          refused([&] { Q4Weights::make<F16>(dev, 64, 128, 32, {}, scales); }) == WKF_ERR_INVALID_ARG && refused([&] { attend(q, cache, 0.125f, true, {4}); }) == WKF_ERR_INVALID_ARG;
      cache.reset();
      std::printf("%s\n", fine && cache.lengths()[0] == 0 ? "OK" : "FAILED");
      return 0;
    }
"""


def test_the_typed_facade_compiles_and_plans(tmp_path):
    gxx, libdir = shutil.which("g++"), os.path.join(ROOT, "wgpu-kernal-fusion_amd")
    if gxx is None:
        pytest.skip("no g++ on this machine")
    (tmp_path / "facade.cpp").write_text(FACADE)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "facade.cpp"), "-o", str(tmp_path / "facade"),
                        "-L", libdir, "-lwkf_hip", f"-Wl,-rpath,{libdir}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(tmp_path / "facade")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


SIBLINGS = r"""
    #include <cstdio>
    #include <wkf_decode.hpp>
    using namespace wkf;
    int main() {
      auto dev = Device::planner();
      Tensor<1, F32> g(dev, {64}, std::vector<float>(64, 1.0f));
      auto table = zeros<2, F32>(dev, {9, 32});
      auto q = norm_rope(zeros<4, F16>(dev, {2, 4, 3, 64}), g, table, table, 1e-5f, {1, 6});
      auto k = norm_rope(zeros<4, F16>(dev, {2, 2, 3, 64}), g, table, table, 1e-5f, {1, 6});
      auto sum = Tensor<1, F32>(dev, {64}, std::vector<float>(64, 2.0f)) + g;
      auto to_q = zeros<4, F16>(dev, {2, 4, 3, 64}), to_k = zeros<4, F16>(dev, {2, 2, 3, 64});
      auto to_sum = zeros<1, F32>(dev, {64});
      materialize_into({{q, to_q}, {k, to_k}});
      const int together = wkf_tensor_kernel_count(q.handle());
      materialize_into({{q, to_q}, {sum, to_sum}, {k, to_k}});
      const int with_sum = wkf_tensor_kernel_count(q.handle());
      int code = 0;
      try { materialize_into({}); } catch (const Error& e) { code = e.code; }
      std::printf("%d %d %d\n", together, with_sum, code);
      return 0;
    }
"""


def test_the_typed_facade_computes_siblings_together(tmp_path, wkf):
    """q and k in one launch, tensors of other ranks and types beside them."""
    gxx, libdir = shutil.which("g++"), os.path.join(ROOT, "wgpu-kernal-fusion_amd")
    if gxx is None:
        pytest.skip("no g++ on this machine")
    (tmp_path / "siblings.cpp").write_text(SIBLINGS)
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "siblings.cpp"), "-o", str(tmp_path / "siblings"),
                        "-L", libdir, "-lwkf_hip", f"-Wl,-rpath,{libdir}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(tmp_path / "siblings")], capture_output=True, text=True, timeout=300)
    counts = r.stdout.split()
    assert r.returncode == 0 and counts[0] == "1" and int(counts[1]) in (2, 3) and counts[2] == str(wkf.ERR_INVALID_ARG), r.stdout + r.stderr
