"""Cases of the training operators next to the pair stack: layer norm with its backward pass,
the global gradient norm with clipping, and the embedding lookup with its gradient by sorted
tokens. Each case runs either as the library's kernels (``own``) or in a plain form written
with elementary torch operations."""

import math
import os
import random
import sys

import torch

own = False  # True: the framework's operators; False: the plain form

EPS = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


_framework = None


def _ops():
    global _framework
    if _framework is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "genie-tk_b200"))
        from genie_tk import ops
        _framework = ops
    return _framework


# --------------------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------------------

def _ln(name, direction, rows, width, dtype="float32", params="float32", grid=0):
    """``grid`` > 0: x is a [grid, grid, width] pair tensor read with its two pair axes swapped."""
    c = {"op": "layernorm", "direction": direction, "rows": grid * grid if grid else rows, "width": width,
         "dtype": dtype, "params": params, "grid": grid}
    return dict(c, name=name) if name else c


def _clip(name, layers, tensors, elements, mix, dtype, out, clipped, pad):
    """``layers`` > 0: the parameter shapes of so many pair-stack layers (four triangle blocks
    and a transition at 128 channels); else ``tensors`` tensors of mixed sizes."""
    c = {"op": "clip", "layers": layers, "tensors": tensors, "elements": elements, "mix": mix, "dtype": dtype,
         "out": out, "clipped": clipped, "pad": pad}
    return dict(c, name=name) if name else c


def _emb(name, direction, tokens, vocab, width, kind, dtype="float32", index="int64", scale=1.0, padding=-1):
    """``kind``: "relative" (the clipped residue offsets of an n x n pair grid, tokens = n * n),
    "zipf" (token frequencies of text) or "uniform" (residue types)."""
    c = {"op": "embedding", "direction": direction, "tokens": tokens, "vocab": vocab, "width": width, "kind": kind,
         "dtype": dtype, "index": index, "scale": scale, "padding": padding}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one short chain's single representation (384 channels): a call that costs its launches
        _ln("layernorm step: short chain", "step", 37, 384),
        # the LayerNorm of every triangle block over the pair tensor, N = 512
        _ln("layernorm forward: pairs", "forward", 0, 128, grid=512),
        # its backward around the ending node, which reads the pair tensor transposed
        _ln("layernorm backward: swapped pairs", "backward", 0, 128, grid=512),
        # a bf16 model's hidden states, a batch of a few thousand tokens
        _ln("layernorm step: hidden states", "step", 4096, 4096, "bfloat16", "bfloat16"),
        # a width that no vector divides, fp16 activations and fp32 parameters
        _ln("layernorm backward: odd width", "backward", 1023, 5003, "float16", "float32"),
        # the gradients of one layer after an ordinary step: below the limit, nothing to scale
        _clip("clip: one layer in place", 1, 0, 0, 0, "float32", "in place", False, 128),
        # an eight-layer stack's gradients clipped into the optimizer's own buffers
        _clip("clip: eight layers", 8, 0, 0, 0, "float32", "same", True, 128),
        # a larger bf16 model: clipped gradients go out in fp32 for the optimizer
        _clip("clip: bf16 to fp32", 0, 200, 1 << 27, 5, "bfloat16", "float32", True, 1),
        # residue types of one chain to its single representation, with the table's gradient
        _emb("embedding step: residues", "step", 300, 21, 384, "uniform"),
        # relative positions of a 512-residue chain into the pair tensor
        _emb("embedding forward: relative positions", "forward", 512 * 512, 66, 128, "relative"),
        # the gradient of that table at 1024 residues: a few rows receive nearly all of the sum
        _emb("embedding backward: relative positions", "backward", 1024 * 1024, 66, 128, "relative"),
        # a vocabulary of subwords in bf16, scaled by sqrt(width), and its gradient
        _emb("embedding step: vocabulary", "step", 8192, 32000, 1024, "zipf", "bfloat16", "int64", 32.0, 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm", "clip", "embedding", "embedding"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "layernorm":
        direction = rng.choice(["forward", "backward", "step"])
        width = _log(rng, 8, 16384)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        most = (1 << 26) // width
        params = rng.choice([dtype, "float32"])
        if rng.random() < 0.3:
            return _ln(None, direction, 0, width, dtype, params, _log(rng, 2, max(2, int(math.sqrt(min(most, 1 << 20))))))
        return _ln(None, direction, _log(rng, 1, min(most, 1 << 21)), width, dtype, params)
    if op == "clip":
        out = rng.choice(["in place", "same", "float32"])
        layers = rng.choice([0, 0, _log(rng, 1, 16)])
        tensors = 0 if layers else _log(rng, 1, 1200)
        elements = 0 if layers else max(tensors, _log(rng, 64, 1 << 26))
        return _clip(None, layers, tensors, elements, rng.randrange(1 << 20), dtype, out,
                     out != "in place" and rng.random() < 0.7, rng.choice([1, 128]))
    direction = rng.choice(["forward", "backward", "step"])
    width = _log(rng, 1, 8192)
    if rng.random() < 0.6:
        width = max(8, width // 8 * 8)
    kind = rng.choice(["relative", "zipf", "uniform"])
    tokens = _log(rng, 1, min((1 << 26) // width, 1 << 20))
    vocab = _log(rng, 2, min((1 << 26) // width, 200000))
    if kind == "relative":
        n = max(1, math.isqrt(tokens))
        tokens, vocab = n * n, 2 * rng.randrange(4, 65) + 2
        width = min(width, 512)
    scale = rng.choice([1.0, math.sqrt(width)])
    return _emb(None, direction, tokens, vocab, width, kind, dtype, rng.choice(["int64", "int32"]), scale,
                rng.choice([-1, 0]))


# --------------------------------------------------------------------------------------
# What a program has in hand before the call
# --------------------------------------------------------------------------------------

def _layer_sizes():
    c, heads, n = 128, 4, 4
    mul = [c, c] + 5 * [c * c, c] + [c * c, c] + [c, c]      # two LayerNorms, six linears with bias
    att = [c, c, heads * c] + 3 * [c * c] + 2 * [c * c, c]   # LayerNorm, bias projection, q, k, v, gate, output
    transition = [c, c, c * n * c, n * c, n * c * c, c]
    return 2 * mul + 2 * att + transition


def _sizes(case):
    if case["layers"]:
        return _layer_sizes() * case["layers"]
    r = random.Random(case["mix"])
    weights = [math.exp(r.uniform(0.0, 8.0)) for _ in range(case["tensors"])]
    total = sum(weights)
    return [max(1, int(case["elements"] * w / total)) for w in weights]


def _offsets(case):
    """Where each gradient begins in the flat buffer, and the buffer's length."""
    at, pad, offsets = 0, case["pad"], []
    for n in _sizes(case):
        offsets.append((at, n))
        at += (n + pad - 1) // pad * pad
    return offsets, at


def _tokens(case, gen, dev):
    t, v, index = case["tokens"], case["vocab"], torch.int64 if case["index"] == "int64" else torch.int32
    if case["kind"] == "relative":
        # offsets j - i of an n x n grid of residues, clipped to +-k; the last token stands for
        # pairs of different chains, and the chain break is somewhere in the middle half
        n, k = math.isqrt(t), (v - 2) // 2
        i = torch.arange(n, device=dev)
        cut = (torch.rand((), generator=gen, device=dev) * 0.5 + 0.25) * n
        chain = i > cut
        tok = (i[None, :] - i[:, None]).clamp(-k, k) + k
        tok = torch.where(chain[None, :] == chain[:, None], tok, torch.full_like(tok, v - 1))
    elif case["kind"] == "zipf":
        u = torch.rand(t, generator=gen, device=dev, dtype=torch.float64)
        tok = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    else:
        tok = torch.randint(0, v, (t,), generator=gen, device=dev)
    return tok.to(index)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "layernorm":
        d, params = case["width"], DTYPES[case["params"]]
        lead = (case["grid"], case["grid"]) if case["grid"] else (case["rows"],)
        x = (randn(*lead, d) * 1.5 + 0.5 * randn(d)).to(dtype)
        dy = (0.01 * randn(*lead, d)).to(dtype)
        if case["grid"]:
            x, dy = x.transpose(0, 1), dy.transpose(0, 1)
        weight, bias = (1.0 + 0.1 * randn(d)).to(params), (0.1 * randn(d)).to(params)
        var, mean = torch.var_mean(x.double(), dim=-1, correction=0)
        return {"case": case, "x": x, "dy": dy, "weight": weight, "bias": bias, "mean": mean.float(),
                "rstd": torch.rsqrt(var + EPS).float()}
    if case["op"] == "clip":
        offsets, length = _offsets(case)
        flat = torch.zeros(length, dtype=dtype, device=dev)
        # layers differ in the size of their gradients: blocks of the buffer at scales of their own
        scales = torch.exp(randn(257) - 6.0)
        at = torch.arange(length, device=dev, dtype=torch.int64) * 257 // length
        values = (randn(length) * scales[at]).to(dtype)
        grads = [flat[a:a + n] for a, n in offsets]
        for (a, n), g in zip(offsets, grads):
            g.copy_(values[a:a + n])
        norm = float(flat.double().square().sum().sqrt())
        out = None
        if case["out"] != "in place":
            out = torch.zeros(length, dtype=dtype if case["out"] == "same" else torch.float32, device=dev)
        outs = None if out is None else [out[a:a + n] for a, n in offsets]
        return {"case": case, "flat": flat, "grads": grads, "out": out, "outs": outs,
                "max_norm": norm * (0.1 if case["clipped"] else 4.0)}
    tok = _tokens(case, gen, dev)
    weight = randn(case["vocab"], case["width"]).to(dtype)
    dy = (0.01 * randn(*tok.shape, case["width"])).to(dtype)
    return {"case": case, "tokens": tok, "weight": weight, "dy": dy}


# --------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------

def _plain_ln_forward(x, weight, bias):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    xc = xf - mean
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + EPS)
    y = (xc * rstd * weight.float() + bias.float()).to(x.dtype)
    return y, mean.squeeze(-1), rstd.squeeze(-1)


def _plain_ln_backward(dy, x, weight, mean, rstd):
    g, rstd = dy.float(), rstd.unsqueeze(-1)
    xhat = (x.float() - mean.unsqueeze(-1)) * rstd
    lead = tuple(range(x.dim() - 1))
    dweight = (g * xhat).sum(lead, dtype=torch.float64).to(weight.dtype)
    dbias = g.sum(lead, dtype=torch.float64).to(weight.dtype)
    g = g * weight.float()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), dweight, dbias


def _layernorm(s):
    x, dy, w, b, direction = s["x"], s["dy"], s["weight"], s["bias"], s["case"]["direction"]
    if own:
        ops = _ops()
        forward, backward = (lambda: ops.layernorm_forward(x, w, b, EPS)), ops.layernorm_backward
    else:
        forward, backward = (lambda: _plain_ln_forward(x, w, b)), _plain_ln_backward
    if direction == "forward":
        return forward()
    if direction == "backward":
        return backward(dy, x, w, s["mean"], s["rstd"])
    y, mean, rstd = forward()
    return (y, *backward(dy, x, w, mean, rstd))


def _clip_run(s):
    if own:
        norm = _ops().clip_grad_norm(s["grads"], s["max_norm"], out=s["outs"])
        return norm, s["flat"] if s["out"] is None else s["out"]
    flat = s["flat"].float()
    norm = flat.square().sum(dtype=torch.float64).sqrt()
    coefficient = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    out = s["flat"] if s["out"] is None else s["out"]
    out.copy_(flat * coefficient)
    return norm.float(), out


def _embedding(s):
    case, tok, w, dy = s["case"], s["tokens"], s["weight"], s["dy"]
    scale, padding = case["scale"], None if case["padding"] < 0 else case["padding"]
    got = []
    if case["direction"] != "backward":
        if own:
            got.append(_ops().embedding_forward(tok, w, scale))
        else:
            got.append((w[tok].float() * scale).to(w.dtype))
    if case["direction"] != "forward":
        if own:
            got.append(_ops().embedding_backward(dy, tok, w.shape[0], scale, padding, w.dtype))
        else:
            # a frequent token's sum runs over up to a million rows: 64 bits
            dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
            dw.index_add_(0, tok.reshape(-1), dy.reshape(-1, w.shape[1]).double())
            if padding is not None:
                dw[padding] = 0.0
            got.append((dw * scale).to(w.dtype))
    return got


def run(state):
    return {"layernorm": _layernorm, "clip": _clip_run, "embedding": _embedding}[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------
# What a pass cannot do without, and its values in 64 bits
# --------------------------------------------------------------------------------------

def _distinct(case):
    """The expected number of different tokens in a call."""
    t, v = case["tokens"], case["vocab"]
    if case["kind"] == "relative":
        return min(t, v)
    if case["kind"] == "uniform":
        return v * -math.expm1(t * math.log1p(-1.0 / v))
    span = math.log(v + 1.0)
    return sum(-math.expm1(t * math.log1p(-math.log((i + 2.0) / (i + 1.0)) / span)) for i in range(v))


def work(case):
    if case["op"] == "layernorm":
        n, e, p = case["rows"] * case["width"], SIZE[case["dtype"]], 2 * case["width"] * SIZE[case["params"]]
        forward = {"bytes": 2 * n * e + 8 * case["rows"] + p, "flops": 7 * n}
        backward = {"bytes": 3 * n * e + 8 * case["rows"] + 3 * p // 2, "flops": 13 * n}
        if case["direction"] == "forward":
            return forward
        if case["direction"] == "backward":
            return backward
        return {k: forward[k] + backward[k] for k in forward}
    if case["op"] == "clip":
        n, e = sum(_sizes(case)), SIZE[case["dtype"]]
        if case["out"] == "in place":  # below the limit: the gradients stay as they are
            return {"bytes": n * e, "flops": 2 * n}
        return {"bytes": n * (e + (e if case["out"] == "same" else 4)), "flops": 3 * n}
    n, e, i = case["tokens"] * case["width"], SIZE[case["dtype"]], 8 if case["index"] == "int64" else 4
    forward = {"bytes": n * e + case["tokens"] * i + _distinct(case) * case["width"] * e, "flops": n}
    backward = {"bytes": n * e + case["tokens"] * i + case["vocab"] * case["width"] * e, "flops": n}
    if case["direction"] == "forward":
        return forward
    if case["direction"] == "backward":
        return backward
    return {k: forward[k] + backward[k] for k in forward}


def _exact_ln_backward(dy, x, w, mean, rstd):
    d = x.shape[-1]
    x, dy = x.reshape(-1, d).double(), dy.reshape(-1, d).double()
    mean, rstd, w = mean.reshape(-1, 1).double(), rstd.reshape(-1, 1).double(), w.double()
    xhat = (x - mean).mul_(rstd)
    db = torch.einsum("rc->c", dy)
    dw = torch.einsum("rc,rc->c", dy, xhat)
    c1 = torch.mv(dy, w) / d
    c2 = torch.einsum("rc,rc,c->r", dy, xhat, w) / d
    dx = dy.mul_(w).sub_(c1[:, None]).addcmul_(xhat, c2[:, None], value=-1.0).mul_(rstd)
    return dx, dw, db


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        x, w, b = s["x"], s["weight"], s["bias"]
        shape = x.shape
        if case["direction"] == "backward":
            dx, dw, db = _exact_ln_backward(s["dy"], x, w, s["mean"], s["rstd"])
            return dx.view(shape), dw, db
        var, mean = torch.var_mean(x.double(), dim=-1, correction=0)
        rstd = (var + EPS).pow(-0.5)
        y = torch.addcmul(b.double(), x.double().sub_(mean.unsqueeze(-1)).mul_(rstd.unsqueeze(-1)), w.double())
        if case["direction"] == "forward":
            return y, mean, rstd
        dx, dw, db = _exact_ln_backward(s["dy"], x, w, mean, rstd)
        return y, dx.view(shape), dw, db
    if case["op"] == "clip":
        flat = s["flat"].double()
        norm = torch.linalg.vector_norm(flat)
        out = flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return norm, out
    tok, w = s["tokens"].long(), s["weight"]
    got = []
    if case["direction"] != "backward":
        got.append(torch.index_select(w, 0, tok.reshape(-1)).double().mul_(case["scale"]).view(*tok.shape, -1))
    if case["direction"] != "forward":
        # sums over runs of equal tokens as differences of one running sum over the sorted rows
        key, order = torch.sort(tok.reshape(-1), stable=True)
        rows = torch.cumsum(s["dy"].reshape(-1, w.shape[1])[order].double(), 0)
        ends = torch.searchsorted(key, torch.arange(w.shape[0], device=key.device), right=True)
        rows = torch.cat([torch.zeros_like(rows[:1]), rows])[ends]
        dw = torch.diff(rows, dim=0, prepend=torch.zeros_like(rows[:1])) * case["scale"]
        if case["padding"] >= 0:
            dw[case["padding"]] = 0.0
        got.append(dw)
    return got
