"""The operators of a decoder's attention block as it serves, case by case: what they are given, their plain form in
elementary torch operations, the framework's own calls, and their values in 64 bits.

  q4         y = x W, W held in 4 bits with a scale (and a zero point) for each group of rows and column
  norm_rope  the root-mean-square norm of every head of q and k, with the rotation of its position
  append     keys and values into a cache of 8 bits, one scale for each block of tokens and head; its values read back
  attend     attention of new tokens over such a cache

`own` chooses between the plain form and the framework.
"""
import functools
import importlib.util
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one token's attention output through a square projection: the latency of a decode step's smallest product
        {"name": "q4 one token", "op": "q4", "dtype": "f16", "m": 1, "k": 4096, "n": 4096, "group": 128, "zeros": False},
        # a few rows kept in f32, with sides that no tile divides and a last group that is not whole
        {"name": "q4 seven rows odd f32", "op": "q4", "dtype": "f32", "m": 7, "k": 4090, "n": 1037, "group": 64, "zeros": True},
        # the gate of a 4096-wide MLP over a prompt
        {"name": "q4 prompt", "op": "q4", "dtype": "f16", "m": 1024, "k": 4096, "n": 11008, "group": 128, "zeros": True},
        # one token of each of 16 sequences, at positions of their own
        {"name": "norm_rope decode", "op": "norm_rope", "dtype": "f16", "batch": 16, "q_heads": 32, "kv_heads": 8, "tokens": 1, "dim": 128, "far": 30000},
        # a prompt of 2048 tokens in f32, as the composites' benchmark has it, with eight key heads
        {"name": "norm_rope prompt f32", "op": "norm_rope", "dtype": "f32", "batch": 1, "q_heads": 32, "kv_heads": 8, "tokens": 2048, "dim": 128, "far": 0},
        # a few tokens of three sequences, the last one with none
        {"name": "append few f32", "op": "append", "dtype": "f32", "batch": 3, "kv_heads": 8, "tokens": 5, "dim": 64, "block": 32, "ragged": True},
        # prompts of four lengths up to 4001
        {"name": "append prompt", "op": "append", "dtype": "f16", "batch": 4, "kv_heads": 8, "tokens": 4001, "dim": 128, "block": 64, "ragged": True},
        # one user, a short conversation: latency
        {"name": "attend one token", "op": "attend", "dtype": "f16", "batch": 1, "q_heads": 32, "kv_heads": 8, "tokens": 1, "length": 1000, "dim": 128, "block": 64, "ragged": False},
        # a serving batch over long caches of many lengths: the bandwidth of the memory
        {"name": "attend batch", "op": "attend", "dtype": "f16", "batch": 16, "q_heads": 32, "kv_heads": 8, "tokens": 1, "length": 32768, "dim": 128, "block": 128, "ragged": True},
        # three tokens at once (a draft to verify) in f32, one query head for each key head, a dimension that is no power of two
        {"name": "attend draft f32", "op": "attend", "dtype": "f32", "batch": 2, "q_heads": 12, "kv_heads": 12, "tokens": 3, "length": 2051, "dim": 80, "block": 32, "ragged": True},
        # the second half of a prompt of 4096 tokens: arithmetic
        {"name": "attend prompt", "op": "attend", "dtype": "f16", "batch": 1, "q_heads": 32, "kv_heads": 8, "tokens": 2048, "length": 4096, "dim": 128, "block": 64, "ragged": False},
        # short prompts of three lengths in f32, the last one empty
        {"name": "attend prompts f32", "op": "attend", "dtype": "f32", "batch": 3, "q_heads": 8, "kv_heads": 8, "tokens": 300, "length": 300, "dim": 64, "block": 64, "ragged": True},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["q4", "norm_rope", "append", "attend", "attend"])
    case = {"op": op, "dtype": rng.choice(["f16", "f16", "f32"])}
    if op == "q4":
        case |= {"m": _log(rng, 1, 1024), "k": _log(rng, 64, 11008), "n": _log(rng, 64, 11008), "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5}
        if rng.random() < 0.5:  # sides as most layers have them
            case |= {"k": -(-case["k"] // 128) * 128, "n": -(-case["n"] // 128) * 128}
        case["m"] = max(1, min(case["m"], 1024 * 4096 * 4096 // (case["k"] * case["n"])))
        return case
    kv_heads = rng.choice([1, 2, 4, 5, 8, 16, 32])
    dim = rng.choice([64, 128, 128, rng.randrange(16, 129, 2), rng.randrange(130, 257, 2)])
    if op == "norm_rope":
        batch, tokens = (1, _log(rng, 1, 2048)) if rng.random() < 0.5 else (_log(rng, 1, 64), 1)
        return case | {"batch": batch, "q_heads": min(32, kv_heads * rng.choice([1, 2, 4, 8])), "kv_heads": kv_heads, "tokens": tokens, "dim": dim, "far": rng.choice([0, 1000, 30000])}
    case |= {"kv_heads": kv_heads, "dim": dim, "block": rng.choice([32, 64, 128]), "ragged": rng.random() < 0.6}
    if op == "append":
        batch = _log(rng, 1, 32)
        return case | {"batch": batch, "tokens": max(1, min(_log(rng, 1, 8192), (1 << 24) // (batch * kv_heads * dim)))}
    case["q_heads"] = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16, 24) if kv_heads * g <= 64])
    if rng.random() < 0.6:  # new tokens of sequences that are under way
        batch, tokens = _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 3, 5])
        length = max(tokens, min(_log(rng, 1, 65536), (1 << 28) // (batch * kv_heads * dim * max(1, case["q_heads"] * tokens // (16 * kv_heads)))))
    else:  # prompts, with or without what was there before
        batch, tokens = _log(rng, 1, 4), _log(rng, 6, 2048)
        tokens = max(6, min(tokens, 2048 * 32 * 64 // (batch * case["q_heads"] * dim)))
        length = tokens + rng.choice([0, 0, _log(rng, 1, 2048)])
    return case | {"batch": batch, "tokens": tokens, "length": length}


# ---- inputs ------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _spread(case, longest):
    """A length for each sequence: all of them, or from `longest` down in equal steps, the last of three or more with none."""
    batch = case["batch"]
    if not case["ragged"] or batch == 1:
        return [longest] * batch
    return [max(1, longest - longest * b // (2 * batch)) if batch < 3 or b < batch - 1 else 0 for b in range(batch)]


def _lengths(case):
    """How long each sequence is with its new tokens, and how many of those it has."""
    if case["op"] == "append":
        counts = _spread(case, case["tokens"])
        return counts, counts
    lengths = _spread(case, case["length"])
    return lengths, [min(n, case["tokens"]) for n in lengths]


def _inputs(case, seed):
    """The inputs of a case, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = DTYPES[case["dtype"]]
    got = {}
    if case["op"] == "q4":
        m, k, n, group = case["m"], case["k"], case["n"], case["group"]
        groups = -(-k // group)
        got["x"] = _normal(gen, m, k).to(kind)
        got["codes"] = torch.clamp(torch.round(_normal(gen, k, n) * 2.6 + 7.5), 0, 15).to(torch.uint8)
        got["scales"] = ((0.5 + torch.rand((groups, n), generator=gen, device="cuda")) * (0.4 / math.sqrt(k))).to(torch.float16)
        got["zeros"] = torch.randint(5, 11, (groups, n), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        return got
    batch, heads, tokens, dim = case["batch"], case["kv_heads"], case["tokens"], case["dim"]
    if case["op"] == "norm_rope":
        # what a projection leaves for its tokens: q heads, then k heads, side by side
        got["qk"] = (_normal(gen, batch, tokens, case["q_heads"] + heads, dim) * 1.5).to(kind)
        got["q_weight"], got["k_weight"] = ((1 + 0.1 * _normal(gen, dim)).to(kind) for _ in range(2))
        got["positions"] = [case["far"] * (b + 1) // batch for b in range(batch)]
        angles = torch.arange(case["far"] + tokens, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        got["cos"], got["sin"] = angles.cos().float(), angles.sin().float()
        return got
    lengths, counts = _lengths(case)
    longest = case["length"] if case["op"] == "attend" else tokens
    # keys as a norm and a rotation leave them, some channels larger than the others; values without
    got["k"] = (_normal(gen, batch, heads, longest, dim) * (0.7 + 0.6 * torch.rand(dim, generator=gen, device="cuda"))).to(kind)
    got["v"] = (_normal(gen, batch, heads, longest, dim) * 0.5).to(kind)
    if case["op"] == "attend":
        got["q"] = _normal(gen, batch, case["q_heads"], tokens, dim).to(kind)
    return got


def _device_list(values, kind=torch.int64):
    return torch.tensor(values, device="cuda", dtype=kind)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["op"] == "append":
        state["counts"] = _device_list(_lengths(case)[1])
    if case["op"] == "norm_rope":
        state["first"] = _device_list(state["positions"])
    if case["op"] == "attend":
        lengths, counts = _lengths(case)
        state["lengths"], state["counts"] = _device_list(lengths), _device_list(counts)
        if not own:  # the cache of a program without the framework: codes and scales
            state["cache"] = [_quantized(state[name], state["lengths"], case["block"]) for name in ("k", "v")]
    if own:
        state = _handed_over(state)
    torch.cuda.synchronize()
    return state


# ---- the plain form ----------------------------------------------------------------------------

def _q4(state):
    group, k = state["case"]["group"], state["case"]["k"]
    zeros = 8.0 if state["zeros"] is None else state["zeros"].float().repeat_interleave(group, 0)[:k]
    weights = (state["codes"].float() - zeros) * state["scales"].float().repeat_interleave(group, 0)[:k]
    return (state["x"].float() @ weights).to(state["x"].dtype)


def _turned(x, weight, cos, sin, first, eps=1e-5):
    """x [batch, tokens, heads, dim] -> [batch, heads, tokens, dim], normalised for each head and rotated."""
    y = x.float()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.float()
    at = first[:, None] + torch.arange(x.shape[1], device=x.device)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    half = x.shape[3] // 2
    low, high = y[..., :half], y[..., half:]
    return torch.cat([low * c - high * s, high * c + low * s], -1).to(x.dtype).transpose(1, 2).contiguous()


def _norm_rope(state):
    heads = state["case"]["q_heads"]
    return {name: _turned(part, state[name + "_weight"], state["cos"], state["sin"], state["first"])
            for name, part in (("q", state["qk"][:, :, :heads]), ("k", state["qk"][:, :, heads:]))}


def _quantized(x, lengths, block):
    """x [batch, heads, tokens, dim] -> codes of 8 bits [batch, heads, blocks, block, dim], and a scale for each block."""
    batch, heads, tokens, dim = x.shape
    blocks = -(-tokens // block)
    there = torch.arange(tokens, device=x.device)[None, :] < lengths[:, None]
    y = torch.zeros((batch, heads, blocks * block, dim), device=x.device, dtype=torch.float32)
    y[:, :, :tokens] = torch.where(there[:, None, :, None], x.float(), 0.0)
    y = y.view(batch, heads, blocks, block, dim)
    largest = y.abs().amax((3, 4))
    scales = largest / torch.full_like(largest, 127.0)  # by a tensor: by a number, torch multiplies with its reciprocal
    # the quotient in 64 bits: in 32, one next to the border of two codes would fall on either side
    codes = (y.double() / scales.double().clamp_min(1e-300)[..., None, None]).round().to(torch.int8)
    return codes, scales


def _values(codes, scales, tokens):
    y = codes.float() * scales[..., None, None]
    return y.flatten(2, 3)[:, :, :tokens]


def _append(state):
    block, tokens = state["case"]["block"], state["case"]["tokens"]
    return torch.stack([_values(*_quantized(state[name], state["counts"], block), tokens) for name in ("k", "v")])


def _attend(state):
    case, q = state["case"], state["q"]
    batch, q_heads, tokens, dim = q.shape
    heads, length = case["kv_heads"], case["length"]
    k, v = (_values(*kept, length) for kept in state["cache"])
    scores = q.float().reshape(batch, heads, -1, dim) @ k.transpose(2, 3) * (1 / math.sqrt(dim))
    scores = scores.view(batch, q_heads, tokens, length)
    row, at = torch.arange(tokens, device=q.device), torch.arange(length, device=q.device)
    last = (state["lengths"] - state["counts"])[:, None] + row  # the row's own place in its sequence
    seen = (at <= last[..., None]) & (row < state["counts"][:, None])[..., None]
    scores = torch.where(seen[:, None], scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(batch, heads, -1, length) @ v).view(batch, q_heads, tokens, dim)
    return torch.where(total > 0, out / total, 0.0).to(q.dtype)


# ---- the framework's calls ---------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _framework():
    """The package (its folder's name is no identifier) and the device, as a program holds them."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wgpu-kernal-fusion_amd", "__init__.py")
    spec = importlib.util.spec_from_file_location("wgpu_kernal_fusion_amd", at)
    package = importlib.util.module_from_spec(spec)
    sys.modules["wgpu_kernal_fusion_amd"] = package
    spec.loader.exec_module(package)
    device = package.Device.new(0)
    device.set_timing(False)
    return package, device


def _room(shape, kind):
    """A tensor of the framework, and torch's view of the same memory."""
    package, device = _framework()
    tensor = package.Tensor.zeros(device, shape, package.F16 if kind == torch.float16 else package.F32)
    return tensor, torch.as_tensor(tensor, device="cuda")


def _given(x):
    tensor, view = _room(tuple(x.shape), x.dtype)
    view.copy_(x)
    return tensor


def _handed_over(state):
    """The same inputs as the framework's tensors, with the weights, the cache and the outputs that a program keeps."""
    package, device = _framework()
    case = state["case"]
    kept = {"case": case}
    if case["op"] == "q4":
        zeros = None if state["zeros"] is None else state["zeros"].cpu().numpy()
        kept["x"] = _given(state["x"])
        kept["weights"] = package.Q4Weights(device, state["codes"].cpu().numpy(), state["scales"].cpu().numpy(), zeros, case["group"])
        kept["out"], kept["view"] = _room((case["m"], case["n"]), state["x"].dtype)
    elif case["op"] == "norm_rope":
        qk, heads = _given(state["qk"]), case["q_heads"]
        kept |= {name: _given(state[name]) for name in ("q_weight", "k_weight", "cos", "sin")}
        kept["positions"] = state["positions"]
        # the heads of q and of k where the projection left them
        kept["parts"] = [qk.narrow(2, 0, heads).transpose(1, 2), qk.narrow(2, heads, case["kv_heads"]).transpose(1, 2)]
        rooms = [_room((case["batch"], n, case["tokens"], case["dim"]), state["qk"].dtype) for n in (heads, case["kv_heads"])]
        kept["outs"], kept["views"] = [r[0] for r in rooms], {"q": rooms[0][1], "k": rooms[1][1]}
    else:
        lengths, counts = _lengths(case)
        kept["counts"] = counts
        kept["k"], kept["v"] = _given(state["k"]), _given(state["v"])
        kept["cache"] = package.KvCache(device, case["batch"], case["kv_heads"], case["dim"], state["k"].shape[2], case["block"])
        torch.cuda.synchronize()
        if case["op"] == "append":
            kept["out"], kept["view"] = _room((2, case["batch"], case["kv_heads"], case["tokens"], case["dim"]), torch.float32)
        else:
            kept["cache"].append(kept.pop("k"), kept.pop("v"), lengths)
            kept["q"] = _given(state["q"])
            kept["out"], kept["view"] = _room(tuple(state["q"].shape), state["q"].dtype)
        device.sync()
    return kept


def _called(state):
    package, _ = _framework()
    case = state["case"]
    if case["op"] == "q4":
        package.materialize_into([state["x"].mat_mul_q4(state["weights"])], [state["out"]])
        return state["view"]
    if case["op"] == "norm_rope":
        turned = [x.norm_rope(state[w], state["cos"], state["sin"], 1e-5, state["positions"]) for x, w in zip(state["parts"], ("q_weight", "k_weight"))]
        package.materialize_into(turned, state["outs"])
        return state["views"]
    if case["op"] == "append":
        state["cache"].reset()
        state["cache"].append(state["k"], state["v"], state["counts"])
        package.materialize_into([state["cache"].values(0, case["tokens"])], [state["out"]])
        return state["view"]
    package.materialize_into([state["q"].attend(state["cache"], 1 / math.sqrt(case["dim"]), True, state["counts"])], [state["out"]])
    return state["view"]


def run(state):
    if own:
        return _called(state)
    return {"q4": _q4, "norm_rope": _norm_rope, "append": _append, "attend": _attend}[state["case"]["op"]](state)


# ---- work and exact values ---------------------------------------------------------------------

def work(case):
    e = 2 if case["dtype"] == "f16" else 4
    if case["op"] == "q4":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": k * n / 2 + -(-k // case["group"]) * n * (2.5 if case["zeros"] else 2) + (m * k + m * n) * e, "flops": 2 * m * k * n}
    batch, heads, tokens, dim = case["batch"], case["kv_heads"], case["tokens"], case["dim"]
    if case["op"] == "norm_rope":
        n = batch * tokens * (case["q_heads"] + heads) * dim
        return {"bytes": 2 * n * e + min(batch * tokens, case["far"] + tokens) * dim * 4 + 2 * dim * e, "flops": 8 * n}
    lengths, counts = _lengths(case)
    if case["op"] == "append":
        return {"bytes": 2 * sum(counts) * heads * dim * e + 2 * batch * tokens * heads * dim * 4, "flops": 4 * sum(counts) * heads * dim}
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lengths, counts))
    blocks = sum(-(-n // case["block"]) for n in lengths)
    return {"bytes": 2 * heads * (sum(lengths) * dim + blocks * 4) + sum(counts) * case["q_heads"] * dim * e + batch * tokens * case["q_heads"] * dim * e,
            "flops": 4 * dim * case["q_heads"] * pairs}


def _stored(x, block):
    """One head's tokens [tokens, dim] as the cache of 8 bits holds them, in 64 bits: the scale is a number of 32 bits."""
    out = torch.empty(x.shape, device=x.device, dtype=torch.float64)
    for part, to in zip(x.double().split(block), out.split(block)):
        scale = (part.abs().max() / 127).float().double()
        to.copy_(torch.round(part / scale) * scale if scale > 0 else part * 0)
    return out


def exact(case, seed):
    """Row by row and head by head, as the definitions are written."""
    got = _inputs(case, seed)
    if case["op"] == "q4":
        x, group = got["x"].double(), case["group"]
        y = torch.zeros((case["m"], case["n"]), device="cuda", dtype=torch.float64)
        for g in range(got["scales"].shape[0]):
            rows = slice(g * group, min(case["k"], (g + 1) * group))
            zero = 8 if got["zeros"] is None else got["zeros"][g].double()
            y += (x[:, rows] @ (got["codes"][rows].double() - zero)) * got["scales"][g].double()
        return y
    if case["op"] == "norm_rope":
        both = {}
        for name, heads in (("q", slice(0, case["q_heads"])), ("k", slice(case["q_heads"], None))):
            x = got["qk"].double().permute(0, 2, 1, 3)[:, heads]
            x = x * (x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-5).pow(-0.5) * got[name + "_weight"].double()
            half = case["dim"] // 2
            for b, first in enumerate(got["positions"]):
                turn = torch.complex(got["cos"].double(), got["sin"].double())[first:first + case["tokens"]]
                pairs = torch.complex(x[b, ..., :half], x[b, ..., half:]) * turn
                x[b] = torch.cat([pairs.real, pairs.imag], -1)
            both[name] = x.contiguous()
        return both
    lengths, counts = _lengths(case)
    if sum(lengths) * case["kv_heads"] / case["block"] > 40000 and case["op"] == "append":
        return None
    if case["op"] == "append":
        y = torch.zeros((2, case["batch"], case["kv_heads"], case["tokens"], case["dim"]), device="cuda", dtype=torch.float64)
        for i, name in enumerate(("k", "v")):
            for b, n in enumerate(lengths):
                for h in range(case["kv_heads"] if n else 0):
                    y[i, b, h, :n] = _stored(got[name][b, h, :n], case["block"])
        return y
    share = case["q_heads"] // case["kv_heads"]
    y = torch.zeros(got["q"].shape, device="cuda", dtype=torch.float64)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        if not n:
            continue
        hidden = torch.ones((c, n), device="cuda").triu(n - c + 1).bool()
        blocks = [got[name][b, :, :n].double() for name in ("k", "v")]
        for i, x in enumerate(blocks):  # whole blocks at once, then what is left
            whole = n // case["block"] * case["block"]
            for part in ([x[:, :whole].unflatten(1, (-1, case["block"]))] if whole else []) + ([x[:, whole:].unsqueeze(1)] if whole < n else []):
                scale = (part.abs().amax((2, 3), keepdim=True) / 127).float().double()
                part.copy_(torch.where(scale > 0, torch.round(part / scale) * scale, 0))
        k, v = blocks
        for h in range(case["q_heads"]):
            score = got["q"][b, h, :c].double() @ k[h // share].T / math.sqrt(case["dim"])
            y[b, h, :c] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[h // share]
    return y


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(8)]:
        print(c, work(c))
