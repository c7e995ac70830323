"""The operators at a decoder's end, and of decoders with layer norm, whose
speed this library is held to: layer norm with its gradients, products of 8-bit
floats with a scale for each block of 128, the distillation loss against a
teacher's top logits with its gradient, and sampling of the next token.

Each case is what a serving loop or a training step does, through the C ABI
(tvk_layer_norm_fwd, tvk_layer_norm_bwd, tvk_gemm_f8, tvk_distill_fwd,
tvk_distill_bwd, tvk_sample) on the current stream, with descriptors the program
keeps over its buffers. The plain forms are the same operators in elementary
torch operations.

Operators (the "op" of a case):
  norm      layer norm after the residual's addition, in the input's type or in
            8 bits with a scale for each block of 128 columns
  norm_bwd  its gradients
  product   x W^T with an 8-bit W and a scale for each 128 x 128 block of it; x
            is 8-bit with a scale for each 128 columns of a row, or is brought
            into that form by the call
  distill   the loss of every row against the teacher's top logits, and its
            gradient
  sample    the next token of every row from its logits and a random number
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1}
F8_MAX = 448.0
EPS = 1e-5
BLOCK = 128


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a few tokens' norm in a decode step, where the launch is all there is
        {"name": "norm_tokens", "op": "norm", "dtype": "fp16", "out": "fp16", "rows": 5, "cols": 1024, "residual": True},
        # a prompt's norm whose output goes to an 8-bit product
        {"name": "norm_prompt_fp8", "op": "norm", "dtype": "bf16", "out": "fp8", "rows": 16384, "cols": 4096,
         "residual": True},
        # a training step's norm, backward
        {"name": "norm_bwd", "op": "norm_bwd", "dtype": "bf16", "rows": 16384, "cols": 2048, "residual": True},
        # ragged rows of a small model, backward
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "dtype": "fp32", "rows": 1000, "cols": 777, "residual": False},
        # one token through a wide layer: the weights' bytes are the time
        {"name": "product_token", "op": "product", "dtype": "bf16", "x": "bf16", "m": 1, "n": 14336, "k": 4096,
         "bias": False},
        # a decode batch, ragged sizes and a bias
        {"name": "product_batch", "op": "product", "dtype": "fp16", "x": "fp16", "m": 50, "n": 5000, "k": 4100,
         "bias": True},
        # a prompt whose norm gave it in 8 bits
        {"name": "product_prompt", "op": "product", "dtype": "bf16", "x": "fp8", "m": 8192, "n": 14336, "k": 4096,
         "bias": False},
        # a training batch against 64 of the teacher's logits
        {"name": "distill", "op": "distill", "dtype": "bf16", "rows": 4096, "cols": 32000, "top": 64, "temperature": 2.0},
        # a short sequence, a ragged vocabulary in 32 bits
        {"name": "distill_short", "op": "distill", "dtype": "fp32", "rows": 33, "cols": 50001, "top": 8,
         "temperature": 1.0},
        # the next token of one sequence
        {"name": "sample_one", "op": "sample", "dtype": "bf16", "rows": 1, "cols": 50001, "spread": 3.0, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "greedy": 0.0, "masked": 0.0},
        # a serving batch with a large vocabulary, no bound on the tokens' number
        {"name": "sample_batch", "op": "sample", "dtype": "bf16", "rows": 64, "cols": 128000, "spread": 3.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "greedy": 0.0, "masked": 0.0},
        # every filter at once, some rows greedy, part of the vocabulary masked, logits in 32 bits
        {"name": "sample_filters", "op": "sample", "dtype": "fp32", "rows": 200, "cols": 32003, "spread": 2.0,
         "top_k": 2000, "top_p": 0.8, "min_p": 0.01, "greedy": 0.1, "masked": 0.2},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, grain=8, odd=0.3):
    """A size between lo and hi, spread over its logarithm: usually a multiple of `grain`, else any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < odd else max(lo, v // grain * grain)


MOST_BYTES = 400e6   # of a drawn case
MOST_FLOPS = 6e11


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "product", "product", "distill", "sample", "sample"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    if op in ("norm", "norm_bwd"):
        cols = _size(rng, 64, 8192)
        rows = max(1, min(_log_int(rng, 1, 16384), int(MOST_BYTES / (4 * cols * BYTES[dtype]))))
        c = {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.6}
        if op == "norm":
            c["out"] = rng.choice([dtype, "fp8"])
        return c
    if op == "product":
        n, k = _size(rng, 200, 16384, 64), _size(rng, 200, 16384, 64)
        m = rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 1, 64), _size(rng, 64, 8192, 16)])
        m = max(1, min(m, int(MOST_FLOPS / (2.0 * n * k))))
        return {"op": op, "dtype": dtype, "x": rng.choice([dtype, "fp8"]), "m": m, "n": n, "k": k,
                "bias": rng.random() < 0.3}
    cols = _size(rng, 1000, 160000, 64)
    if op == "distill":
        rows = max(1, min(_log_int(rng, 1, 8192), int(MOST_BYTES / (2 * cols * BYTES[dtype]))))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "top": _log_int(rng, 1, 256),
                "temperature": rng.choice([1.0, 1.0, 2.0, 0.7, 4.0])}
    return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 256), "cols": cols,
            "spread": rng.choice([1.0, 2.0, 3.0, 4.0]), "top_k": rng.choice([0, 0, 1, 20, 50, 200, 5000]),
            "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.0, 0.02, 0.1]),
            "greedy": rng.choice([0.0, 0.0, 0.2]), "masked": rng.choice([0.0, 0.0, 0.3, 0.99])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _Source:
    """Seeded values made on the GPU, rounded to the case's type."""

    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))
        self.dtype = DTYPES[case["dtype"]]

    def __call__(self, *shape, std=1.0, dtype=None):
        x = torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32)
        return (x * std if std != 1.0 else x).to(dtype or self.dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=torch.float32)


def _blocks(n):
    return -(-n // BLOCK)


def _in_blocks(x, tall):
    """x [rows, cols] in float32 as (8-bit values, scale of each block of `tall` rows and 128 columns)."""
    rows, cols = x.shape
    padded = torch.zeros((-(-rows // tall) * tall, _blocks(cols) * BLOCK), dtype=torch.float32, device="cuda")
    padded[:rows, :cols] = x
    tiles = padded.view(-1, tall, _blocks(cols), BLOCK)
    top = tiles.abs().amax((1, 3))
    scale = torch.where(top > 0, top / F8_MAX, 1.0)
    q = _in8(tiles / scale[:, None, :, None]).view(torch.uint8).view(padded.shape)[:rows, :cols]
    return q.contiguous().view(torch.float8_e4m3fn), scale


def _inputs(case, seed):
    c, r = case, _Source(case, seed)
    if c["op"] in ("norm", "norm_bwd"):
        d = {"w": r(c["cols"], std=0.2) + 1}
        if c["op"] == "norm":
            d["b"] = r(c["cols"], std=0.2)
            d["x"] = r(c["rows"], c["cols"])
            if c["residual"]:
                d["r"] = r(c["rows"], c["cols"], std=2.0)
        else:
            d["h"], d["dy"] = r(c["rows"], c["cols"], std=2.0) + 0.5, r(c["rows"], c["cols"])
            if c["residual"]:
                d["dh"] = r(c["rows"], c["cols"])
        return d
    if c["op"] == "product":
        d = dict(zip(("w", "w_scale"), _in_blocks(r(c["n"], c["k"], std=c["k"] ** -0.5, dtype=torch.float32), BLOCK)))
        # activations whose columns are of unlike size, which is what the blocks' scales are for
        x = r(c["m"], c["k"], dtype=torch.float32) * torch.exp(r(c["k"], dtype=torch.float32))
        if c["x"] == "fp8":
            d["x"], d["x_scale"] = _in_blocks(x, 1)
        else:
            d["x"] = x.to(DTYPES[c["x"]])
        if c["bias"]:
            d["bias"] = r(c["n"])
        return d
    if c["op"] == "distill":
        d = {"logits": r(c["rows"], c["cols"], std=3.0)}
        noisy = d["logits"].float().add_(r(c["rows"], c["cols"], dtype=torch.float32))
        top, index = noisy.topk(min(c["top"], c["cols"]), -1)
        # lists are of unlike length, every seventeenth position is padding, and some lists name an index twice
        length = (r.uniform(c["rows"], 1) * c["top"]).long() // 2 + (c["top"] + 1) // 2
        length[16::17] = 0
        index = torch.where(torch.arange(c["top"], device="cuda") < length, index, -1)
        if c["top"] > 2:
            index[::5, 2] = index[::5, 0]
        d["teacher"], d["index"] = top.contiguous(), index.contiguous()
        d["dloss"] = r.uniform(c["rows"]) / c["rows"]
        return d
    rows, cols = c["rows"], c["cols"]
    logits = r(rows, cols, std=c["spread"])
    if c["masked"]:
        logits.masked_fill_(r.uniform(rows, cols) < c["masked"], float("-inf"))
    d = {"logits": logits, "random": r.uniform(rows)}
    d["temperature"] = 0.5 + r.uniform(rows)
    if c["greedy"]:
        d["temperature"] = torch.where(r.uniform(rows) < c["greedy"], 0.0, d["temperature"])
    if c["top_k"]:
        d["top_k"] = (c["top_k"] * (1 + r.uniform(rows)) / 2).ceil().to(torch.int32)
    if c["top_p"] < 1:
        d["top_p"] = c["top_p"] + (1 - c["top_p"]) * r.uniform(rows) / 2
    if c["min_p"]:
        d["min_p"] = c["min_p"] * (0.5 + r.uniform(rows))
    return d


# ---------------------------------------------------------------------------
# prepare and run
# ---------------------------------------------------------------------------

class _State:
    """A case's tensors and, for the library's calls, the descriptors over them and the buffers they write."""

    def __init__(self, case, tensors):
        self.case, self.t, self.calls, self.out = case, tensors, None, None


def _describe(s):
    """The descriptors that a program keeps over its buffers."""
    from torchvulkan_amd import _abi

    c, t = s.case, s.t
    stream = torch.cuda.current_stream().cuda_stream

    def empty(*shape, dtype=DTYPES[c["dtype"]]):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if c["op"] == "norm":
        y = empty(c["rows"], c["cols"], dtype=DTYPES[c["out"]])
        h = torch.empty_like(t["x"]) if c["residual"] else None
        scale = empty(c["rows"], _blocks(c["cols"]), dtype=torch.float32) if c["out"] == "fp8" else None
        made = [("tvk_layer_norm_fwd", _abi.make_layer_norm_desc(t["x"], t["w"], t["b"], y, residual=t.get("r"),
                                                                residual_out=h, scale=scale, eps=EPS, stream=stream))]
        s.out = {"y": y, "h": h, "scale": scale}
    elif c["op"] == "norm_bwd":
        dx, dw, db = torch.empty_like(t["h"]), torch.empty_like(t["w"]), torch.empty_like(t["w"])
        made = [("tvk_layer_norm_bwd", _abi.make_layer_norm_bwd_desc(t["dy"], t["h"], t["w"], dx, dw, db, dh=t.get("dh"),
                                                                    eps=EPS, stream=stream))]
        s.out = {"dx": dx, "dw": dw, "db": db}
    elif c["op"] == "product":
        y = empty(c["m"], c["n"])
        made = [("tvk_gemm_f8", _abi.make_gemm_f8_desc(t["x"], t.get("x_scale"), t["w"], t["w_scale"], y,
                                                      bias=t.get("bias"), stream=stream))]
        s.out = {"y": y}
    elif c["op"] == "distill":
        loss, lse = empty(c["rows"], dtype=torch.float32), empty(c["rows"], dtype=torch.float32)
        target, grad = empty(c["rows"], c["top"], dtype=torch.float32), torch.empty_like(t["logits"])
        made = [("tvk_distill_fwd", _abi.make_distill_desc(t["logits"], t["index"], t["teacher"], loss, lse, target,
                                                          temperature=c["temperature"], stream=stream)),
                ("tvk_distill_bwd", _abi.make_distill_bwd_desc(t["logits"], t["index"], lse, target, t["dloss"], grad,
                                                              temperature=c["temperature"], stream=stream))]
        s.out = {"loss": loss, "dlogits": grad}
    else:
        token, logprob = empty(c["rows"], dtype=torch.int64), empty(c["rows"], dtype=torch.float32)
        made = [("tvk_sample", _abi.make_sample_desc(t["logits"], t["random"], token, logprob, t["temperature"],
                                                    t.get("top_k"), t.get("top_p"), t.get("min_p"), stream=stream))]
        s.out = {"token": token, "logprob": logprob}
    s.calls = [(getattr(_abi.load(), fn), ctypes.byref(d), _abi.check) for fn, d in made]


def prepare(case, seed):
    s = _State(case, _inputs(case, seed))
    if own:
        _describe(s)
    return s


def run(state):
    if own:
        for fn, desc, check in state.calls:
            status = fn(desc)
            if status:
                check(status)
        return state.out
    return {"norm": _norm, "norm_bwd": _norm_bwd, "product": _product, "distill": _distill, "sample": _sample}[
        state.case["op"]](state.case, state.t)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _in8(x):
    return x.clamp(-F8_MAX, F8_MAX).to(torch.float8_e4m3fn)


def _norm(c, t):
    h = t["x"]
    if c["residual"]:
        h = (t["x"].float() + t["r"].float()).to(h.dtype)
    x = h.float()
    x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * t["w"].float() + t["b"].float()
    y, scale = _in_blocks(y, 1) if c["out"] == "fp8" else (y.to(h.dtype), None)
    return {"y": y, "h": h if c["residual"] else None, "scale": scale}


def _norm_bwd(c, t):
    h, dy, w = t["h"].float(), t["dy"].float(), t["w"].float()
    x = h - h.mean(-1, keepdim=True)
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * inv
    g = dy * w
    dx = inv * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if c["residual"]:
        dx = dx + t["dh"].float()
    return {"dx": dx.to(t["h"].dtype), "dw": (dy * n).sum(0).to(t["w"].dtype), "db": dy.sum(0).to(t["w"].dtype)}


def _spread(scale, tall, rows, cols):
    """Each block's scale at each of its places."""
    return scale.repeat_interleave(tall, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _product(c, t):
    x, scale = (t["x"], t["x_scale"]) if c["x"] == "fp8" else _in_blocks(t["x"].float(), 1)
    x = x.float() * _spread(scale, 1, c["m"], c["k"])
    w = t["w"].float() * _spread(t["w_scale"], BLOCK, c["n"], c["k"])
    y = torch.matmul(x, w.t())
    if c["bias"]:
        y = y + t["bias"].float()
    return {"y": y.to(DTYPES[c["dtype"]])}


def _distill(c, t):
    temperature = c["temperature"]
    s = t["logits"].float() / temperature
    s = s - s.amax(-1, keepdim=True)
    logp = s - s.exp().sum(-1, keepdim=True).log()
    named = t["index"] >= 0
    index = t["index"].clamp(min=0)
    q = (t["teacher"].float() / temperature).masked_fill(~named, float("-inf"))
    top = q.amax(-1, keepdim=True)
    q = q - torch.where(top == float("-inf"), 0.0, top)
    logq = q - q.exp().sum(-1, keepdim=True).log()
    q = torch.where(named, logq.exp(), 0.0)
    loss = torch.where(q > 0, q * (logq - logp.gather(1, index)), 0.0).sum(-1) * temperature ** 2
    grad = torch.where(named.any(-1, keepdim=True), logp.exp(), 0.0).scatter_add_(1, index, -q)
    grad = grad * (t["dloss"] * temperature)[:, None]
    return {"loss": loss, "dlogits": grad.to(t["logits"].dtype)}


def _sample(c, t):
    """In 64 bits: which token is drawn turns on sums that end next to a border."""
    logits, rows, cols = t["logits"].double(), c["rows"], c["cols"]
    greedy = t["temperature"] <= 0
    temperature = torch.where(greedy, 1.0, t["temperature"].double())[:, None]
    value, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    rank = torch.arange(cols, device="cuda")
    w = torch.exp((value - value[:, :1]) / temperature)
    keep = (w > 0) & (rank < torch.where(greedy, 1, cols)[:, None])
    if "top_k" in t:
        keep &= rank < t["top_k"][:, None]
    w = torch.where(keep, w, 0.0)
    if "top_p" in t:
        total = w.cumsum(-1)
        keep &= total - w < t["top_p"].double()[:, None] * total[:, -1:]
    if "min_p" in t:
        keep &= w >= t["min_p"].double()[:, None]
    keep[:, 0] = True
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(kept, torch.exp((logits - value[:, :1]) / temperature), 0.0)
    total = w.cumsum(-1)
    token = (total <= t["random"].double()[:, None] * total[:, -1:]).sum(-1).clamp(max=cols - 1)
    logprob = torch.log(w.gather(1, token[:, None]) / total[:, -1:])[:, 0]
    return {"token": token, "logprob": logprob.float()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, e = case, BYTES[case["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["cols"]
        out = BYTES[c["out"]]
        return {"bytes": n * ((3 if c["residual"] else 1) * e + out) + 2 * c["cols"] * e
                + (4 * c["rows"] * _blocks(c["cols"]) if out == 1 else 0), "flops": (8 if c["residual"] else 7) * n}
    if c["op"] == "norm_bwd":
        n = c["rows"] * c["cols"]
        return {"bytes": n * e * (4 if c["residual"] else 3) + 3 * c["cols"] * e, "flops": 15 * n}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        x = m * k * BYTES[c["x"]] + (4 * m * _blocks(k) if c["x"] == "fp8" else 0)
        return {"bytes": x + n * k + 4 * _blocks(n) * _blocks(k) + m * n * e + (n * e if c["bias"] else 0),
                "flops": 2 * m * n * k}
    n = c["rows"] * c["cols"]
    if c["op"] == "distill":
        return {"bytes": 2 * n * e + c["rows"] * (12 * c["top"] + 8), "flops": 8 * n}
    return {"bytes": n * e + 32 * c["rows"], "flops": 4 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _e4m3(x):
    """x on the e4m3 grid, nearest, ties to the even step."""
    x = x.clamp(-F8_MAX, F8_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_rows_in_blocks(x):
    """x [rows, cols] in 64 bits: 8-bit values and the scale of each 128 columns of a row."""
    q, scales = torch.empty_like(x), []
    for first in range(0, x.shape[1], BLOCK):
        part = x[:, first:first + BLOCK]
        scale = part.abs().max(-1, keepdim=True).values / F8_MAX
        scale[scale == 0] = 1
        q[:, first:first + BLOCK] = _e4m3(part / scale)
        scales.append(scale)
    return q, torch.cat(scales, 1)


def _exact_norm(c, t):
    h = t["x"].double()
    if c["residual"]:
        h = (h + t["r"].double()).to(t["x"].dtype).double()
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    y = (h - mean) / torch.sqrt(var + EPS) * t["w"].double() + t["b"].double()
    y, scale = _exact_rows_in_blocks(y) if c["out"] == "fp8" else (y, None)
    return {"y": y, "h": h if c["residual"] else None, "scale": scale}


def _exact_norm_bwd(c, t):
    h, dy, n = t["h"].double(), t["dy"].double(), c["cols"]
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    sd = (var + EPS).sqrt()
    x, g = h - mean, dy * t["w"].double()
    dx = (g - g.sum(-1, keepdim=True) / n) / sd - x * (g * x).sum(-1, keepdim=True) / (n * sd ** 3)
    if c["residual"]:
        dx = dx + t["dh"].double()
    return {"dx": dx, "dw": (dy * x / sd).sum(0), "db": dy.sum(0)}


def _exact_product(c, t):
    if c["x"] == "fp8":
        q, scale = t["x"].double(), t["x_scale"].double()
    else:
        q, scale = _exact_rows_in_blocks(t["x"].double())
    y = torch.zeros((c["m"], c["n"]), dtype=torch.float64, device="cuda")
    for i, first in enumerate(range(0, c["k"], BLOCK)):
        w = t["w"][:, first:first + BLOCK].double() * t["w_scale"][:, i].double().repeat_interleave(BLOCK)[:c["n"], None]
        y += (q[:, first:first + BLOCK] * scale[:, i:i + 1]) @ w.t().contiguous()
    if c["bias"]:
        y += t["bias"].double()
    return {"y": y}


def _exact_distill(c, t):
    loss = torch.zeros(c["rows"], dtype=torch.float64, device="cuda")
    grad = torch.zeros((c["rows"], c["cols"]), dtype=torch.float64, device="cuda")
    index, teacher, heat = t["index"].cpu(), t["teacher"], c["temperature"]
    for row in range(c["rows"]):
        named = (index[row] >= 0).nonzero()[:, 0]
        if not len(named):
            continue
        at = index[row][named].cuda()
        logp = torch.log_softmax(t["logits"][row].double() / heat, -1)
        logq = torch.log_softmax(teacher[row][named.cuda()].double() / heat, -1)
        loss[row] = heat * heat * (logq.exp() * (logq - logp[at])).sum()
        grad[row] = logp.exp().index_add_(0, at, -logq.exp()) * (heat * t["dloss"][row].double())
    return {"loss": loss, "dlogits": grad}


def _exact_sample(c, t):
    tokens, logprobs = [], []
    read = {name: t[name].cpu().double().tolist() for name in ("random", "temperature", "top_k", "top_p", "min_p") if name in t}
    for row in range(c["rows"]):
        l = t["logits"][row].double()
        l = l + 0.0
        heat = read["temperature"][row]
        best = l.max()
        if heat <= 0:
            tokens.append(int((l == best).nonzero()[0]))
            logprobs.append(0.0)
            continue
        w = torch.exp((l - best) / heat)
        # places from the largest on, of equal ones the first before the later
        places = torch.argsort(-l, stable=True)
        places = places[:min(int((w > 0).sum()), int(read["top_k"][row]) if "top_k" in read else c["cols"])]
        if "top_p" in read:
            sums = torch.cumsum(w[places], 0)
            places = places[:int((sums < read["top_p"][row] * sums[-1]).sum()) + 1]
        if "min_p" in read:
            places = places[:max(1, int((w[places] >= read["min_p"][row]).sum()))]
        places = torch.sort(places).values
        sums = torch.cumsum(w[places], 0)
        i = int(torch.searchsorted(sums, read["random"][row] * sums[-1:], right=True))
        place = places[min(i, len(places) - 1)]
        tokens.append(int(place))
        logprobs.append(float(torch.log(w[place] / sums[-1])))
    return {"token": torch.tensor(tokens), "logprob": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    t = _inputs(case, seed)
    return {"norm": _exact_norm, "norm_bwd": _exact_norm_bwd, "product": _exact_product, "distill": _exact_distill,
            "sample": _exact_sample}[case["op"]](case, t)
