"""The decoder-block operators whose speed this library is held to: a paged
key/value cache (append with rotation, attention) and the root-mean-square norm.

Each case is one call that a serving loop or a training step makes, through the
C ABI (tvk_paged_append, tvk_paged_attention, tvk_rms_norm_fwd,
tvk_rms_norm_bwd) on the current stream, with a descriptor the program keeps
over its buffers. The plain forms are the same operators in elementary torch
operations.

Operators (the "op" of a case):
  append     rotates the new tokens' queries and keys by their positions and
             writes keys and values into their pages
  attention  attention of each sequence's newest tokens over its pages
  norm       root-mean-square norm after the residual's addition, in the
             input's type or in 8 bits with a scale for each row
  norm_bwd   its gradients
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


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

# lengths of a batch: the longest is "len", the shortest "low" of it, the others evenly between; the last "idle" slots of
# the batch hold no sequence (length 0), as a batch of fixed size has them

def listed():
    return [
        # the smallest call of a decode step: one token of one sequence, where the launch is all there is
        {"name": "append_token", "op": "append", "dtype": "fp16", "cache": "fp16", "batch": 1, "new": 1, "hq": 8,
         "hkv": 2, "dim": 64, "rot": 64, "pairs": False, "page": 16, "order": "slots", "len": 300, "low": 1.0, "idle": 0},
        # four prompts of 2048 tokens filling their pages
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "cache": "bf16", "batch": 4, "new": 2048, "hq": 32,
         "hkv": 8, "dim": 128, "rot": 128, "pairs": False, "page": 64, "order": "slots", "len": 2500, "low": 0.85,
         "idle": 0},
        # five drafted tokens for each sequence of a serving batch, into a cache held in 8 bits
        {"name": "append_drafts_fp8", "op": "append", "dtype": "bf16", "cache": "fp8", "batch": 48, "new": 5, "hq": 32,
         "hkv": 8, "dim": 128, "rot": 64, "pairs": True, "page": 32, "order": "heads", "len": 1000, "low": 0.1,
         "idle": 3},
        # two short sequences of a small decoder, where latency counts
        {"name": "attend_short", "op": "attention", "dtype": "fp16", "cache": "fp16", "batch": 2, "new": 1, "hq": 8,
         "hkv": 2, "dim": 64, "page": 16, "order": "slots", "len": 200, "low": 0.5, "idle": 0, "window": 0},
        # a serving batch whose sequences have very different lengths
        {"name": "attend_batch", "op": "attention", "dtype": "bf16", "cache": "bf16", "batch": 32, "new": 1, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "order": "slots", "len": 8000, "low": 0.1, "idle": 2, "window": 0},
        # one long document: the cache's length is all the parallelism there is
        {"name": "attend_long", "op": "attention", "dtype": "bf16", "cache": "bf16", "batch": 1, "new": 1, "hq": 32,
         "hkv": 8, "dim": 128, "page": 128, "order": "heads", "len": 100001, "low": 1.0, "idle": 0, "window": 0},
        # drafted tokens checked over a cache held in 8 bits
        {"name": "attend_drafts_fp8", "op": "attention", "dtype": "bf16", "cache": "fp8", "batch": 24, "new": 4,
         "hq": 32, "hkv": 8, "dim": 128, "page": 32, "order": "slots", "len": 6001, "low": 0.2, "idle": 0, "window": 0},
        # no shared heads, a head dimension that is no power of two, pages of an odd count, a sliding window
        {"name": "attend_window_odd", "op": "attention", "dtype": "fp16", "cache": "fp16", "batch": 16, "new": 1,
         "hq": 12, "hkv": 12, "dim": 80, "page": 20, "order": "slots", "len": 3001, "low": 0.1, "idle": 1,
         "window": 1000},
        # a few tokens' norm in a decode step
        {"name": "norm_tokens", "op": "norm", "dtype": "fp16", "out": "fp16", "rows": 7, "cols": 4096, "residual": True},
        # a prompt's norm whose output goes to an 8-bit product
        {"name": "norm_prompt_fp8", "op": "norm", "dtype": "bf16", "out": "fp8", "rows": 16384, "cols": 4096,
         "residual": True},
        # a training step's norm, backward
        {"name": "norm_bwd", "op": "norm_bwd", "dtype": "bf16", "rows": 16384, "cols": 2048, "residual": True},
        # ragged rows of a small model, backward
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "dtype": "fp16", "rows": 1000, "cols": 777, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, grain=8, odd=0.3):
    """A size between lo and hi, spread over its logarithm: usually a multiple of `grain`, else any number."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < odd else max(lo, v // grain * grain)


MOST_BYTES = 400e6   # of a drawn case


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "norm", "norm_bwd"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp16", "bf16", "fp32"])
    if op in ("norm", "norm_bwd"):
        cols = _size(rng, 64, 8192)
        rows = max(1, min(_log_int(rng, 1, 16384), int(MOST_BYTES / (4 * cols * BYTES[dtype]))))
        c = {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.6}
        if op == "norm":
            c["out"] = rng.choice([dtype, "fp8"])
        return c
    hkv = rng.choice([1, 2, 4, 8, 16])
    hq = min(64, hkv * rng.choice([1, 2, 4, 4, 8, 16]))
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([1, 16, 16, 32, 64, 128, 256, 20, 48])
    cache = dtype if dtype == "fp32" else rng.choice([dtype, dtype, "fp8"])
    c = {"op": op, "dtype": dtype, "cache": cache, "hq": hq, "hkv": hkv, "dim": dim, "page": page,
         "order": rng.choice(["slots", "heads"]), "low": rng.choice([1.0, 0.5, 0.1, 0.02])}
    if op == "append":
        c["new"] = rng.choice([1, 1, 2, 5, _size(rng, 16, 2048, 16)])
        token = (hq + hkv) * dim * 2 * BYTES[dtype]
        c["batch"] = max(1, min(_log_int(rng, 1, 128), int(MOST_BYTES / (token * c["new"]))))
        c["rot"] = rng.choice([dim, dim, dim // 2])
        c["pairs"] = rng.random() < 0.3
        slot = hkv * dim * c["batch"]
        c["len"] = c["new"] + rng.randrange(0, max(1, min(4000, (1 << 25) // slot)))
    else:
        c["new"] = rng.choice([1, 1, 1, 1, 2, 4, 8])
        c["len"] = max(c["new"], _size(rng, 1, 65536, 64, 0.7))
        slot = hkv * dim * 2 * BYTES[cache]
        if dtype == "fp32":
            c["len"] = min(c["len"], 4096)
        c["len"] = max(c["new"], min(c["len"], int(MOST_BYTES / slot)))
        c["batch"] = max(1, min(_log_int(rng, 1, 128), int(MOST_BYTES / (slot * c["len"])),
                                (1 << 27) // (c["len"] * hkv * dim)))
        c["window"] = _size(rng, 32, 4096, 32) if rng.random() < 0.2 else 0
    c["idle"] = rng.choice([0, 0, 1]) if c["batch"] > 1 else 0
    return c


def _lens(c):
    """The batch's lengths before they are put in an order."""
    live = c["batch"] - c["idle"]
    low = max(1, int(c["low"] * c["len"]))
    return [c["len"] - (c["len"] - low) * i // max(1, live - 1) for i in range(live)] + [0] * c["idle"]


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

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def uniform(self, n, lo, hi):
        return lo + (hi - lo) * torch.rand((n,), generator=self.g, device="cuda", dtype=torch.float32)


def _frequencies(rot):
    """Angle of one position for each rotated pair."""
    return torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(0, rot, 2, dtype=torch.float64) / rot)


def _cached(c, r):
    """A paged cache, and where each sequence's pages are: pages in an order of their own, -1 past a sequence's last."""
    lens = torch.tensor(_lens(c), dtype=torch.int64, device="cuda")[r.perm(c["batch"])]
    need = (lens + c["page"] - 1) // c["page"]
    pages, width = int(need.sum()), max(1, int(need.max()))
    at = torch.arange(width, device="cuda")
    first = torch.cumsum(need, 0) - need
    held = at[None, :] < need[:, None]
    order = torch.cat([r.perm(pages), torch.zeros(1, dtype=torch.int64, device="cuda")])
    table = torch.where(held, order[torch.where(held, first[:, None] + at, pages)], -1).to(torch.int32)
    # one page more than the sequences hold, where tokens without a place may be put
    shape = (pages + 1, c["page"], c["hkv"], c["dim"]) if c["order"] == "slots" else \
        (pages + 1, c["hkv"], c["page"], c["dim"])
    d = {"lens": lens.to(torch.int32), "table": table.contiguous()}
    for name in ("k", "v"):
        cache = r(*shape, dtype=DTYPES[c["cache"]])
        # [page, slot, head, dim] whatever the order underneath
        d[name + "_cache"] = cache if c["order"] == "slots" else cache.transpose(1, 2)
        if c["cache"] == "fp8":
            d[name + "_scale"] = r.uniform(c["hkv"], 0.25, 2.0)
    return d


def _inputs(case, seed):
    c, r = case, _Source(case, seed)
    if c["op"] in ("append", "attention"):
        d = _cached(c, r)
        # one projection's output holds queries, keys and values side by side
        heads = r(c["batch"], c["new"], c["hq"] + 2 * c["hkv"], c["dim"])
        d["q"], d["k"], d["v"] = heads.split([c["hq"], c["hkv"], c["hkv"]], dim=2)
        if c["op"] == "append" and c["rot"]:
            angle = torch.arange(c["len"], dtype=torch.float64)[:, None] * _frequencies(c["rot"])
            d["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        return d
    d = {"w": r(c["cols"], std=0.2) + 1}
    if c["op"] == "norm":
        d["x"] = r(c["rows"], c["cols"])
        if c["residual"]:
            d["r"] = r(c["rows"], c["cols"], std=2.0)
    else:
        d["h"], d["dy"] = r(c["rows"], c["cols"], std=2.0), r(c["rows"], c["cols"])
        if c["residual"]:
            d["dh"] = r(c["rows"], c["cols"])
    return d


# ---------------------------------------------------------------------------
# prepare and run
# ---------------------------------------------------------------------------

class _State:
    """A case's tensors and, for the library's calls, the descriptor over them and the buffers it writes."""

    def __init__(self, case, tensors):
        self.case, self.t, self.call, self.out = case, tensors, None, None


def _describe(s):
    """The descriptor that a program keeps over its buffers."""
    from torchvulkan_amd import _abi

    c, t = s.case, s.t
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        # queries are rotated into a buffer of their own, so that a call can be made again
        q_out = torch.empty(t["q"].shape, dtype=t["q"].dtype, device="cuda")
        d = _abi.make_paged_append_desc(t["q"], t["k"], t["v"], q_out, t["k_cache"][:-1], t["v_cache"][:-1], t["lens"],
                                        t["table"], rotary=t.get("rotary"), interleaved=c["pairs"],
                                        k_scale=t.get("k_scale"), v_scale=t.get("v_scale"), stream=stream)
        out, fn = {"q": q_out, "k_cache": t["k_cache"][:-1], "v_cache": t["v_cache"][:-1]}, "tvk_paged_append"
    elif c["op"] == "attention":
        o = torch.empty(t["q"].shape, dtype=t["q"].dtype, device="cuda")
        d = _abi.make_paged_attention_desc(t["q"], t["k_cache"][:-1], t["v_cache"][:-1], o, t["lens"], t["table"],
                                           max_len=c["len"], window=c["window"], k_scale=t.get("k_scale"),
                                           v_scale=t.get("v_scale"), stream=stream)
        out, fn = {"out": o}, "tvk_paged_attention"
    elif c["op"] == "norm":
        y = torch.empty(t["x"].shape, dtype=DTYPES[c["out"]], device="cuda")
        h = torch.empty_like(t["x"]) if c["residual"] else None
        scale = torch.empty(c["rows"], dtype=torch.float32, device="cuda") if c["out"] == "fp8" else None
        d = _abi.make_rms_norm_desc(t["x"], t["w"], y, residual=t.get("r"), residual_out=h, scale=scale, eps=EPS,
                                    stream=stream)
        out, fn = {"y": y, "h": h, "scale": scale}, "tvk_rms_norm_fwd"
    else:
        dx, dw = torch.empty_like(t["h"]), torch.empty_like(t["w"])
        d = _abi.make_rms_norm_bwd_desc(t["dy"], t["h"], t["w"], dx, dw, dh=t.get("dh"), eps=EPS, stream=stream)
        out, fn = {"dx": dx, "dw": dw}, "tvk_rms_norm_bwd"
    s.call, s.out = (getattr(_abi.load(), fn), ctypes.byref(d), _abi.check), out


def prepare(case, seed):
    s = _State(case, _inputs(case, seed))
    if own:
        _describe(s)
    return s


def run(state):
    if own:
        fn, desc, check = state.call
        status = fn(desc)
        if status:
            check(status)
        return state.out
    return {"append": _append, "attention": _attention, "norm": _norm, "norm_bwd": _norm_bwd}[state.case["op"]](
        state.case, state.t)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _in8(x):
    return x.clamp(-F8_MAX, F8_MAX).to(torch.float8_e4m3fn)


def _rotate(x, cos, sin, pairs):
    """x [B, T, H, D] with its first 2 * cos.shape[-1] values of each head rotated."""
    half = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if pairs:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _places(c, t):
    """Position, page and slot of every new token; tokens without a place go to the last page."""
    pos = t["lens"][:, None].long() - c["new"] + torch.arange(c["new"], device="cuda")
    fits = pos >= 0
    at = pos.clamp(min=0)
    page = torch.gather(t["table"].long(), 1, at // c["page"])
    spare = t["k_cache"].shape[0] - 1
    return at, fits, torch.where(fits, page, spare), at % c["page"]


def _append(c, t):
    at, fits, page, slot = _places(c, t)
    q, k, v = t["q"].float(), t["k"].float(), t["v"].float()
    if "rotary" in t:
        cos, sin = t["rotary"][at].chunk(2, -1)
        q, k = _rotate(q, cos, sin, c["pairs"]), _rotate(k, cos, sin, c["pairs"])
    q = torch.where(fits[:, :, None, None], q, 0.0)
    for name, x in (("k", k), ("v", v)):
        cache = t[name + "_cache"]
        if c["cache"] == "fp8":
            x, cache = _in8(x / t[name + "_scale"][:, None]).view(torch.uint8), cache.view(torch.uint8)
        cache[page, slot] = x.to(cache.dtype)
    return {"q": q.to(t["q"].dtype), "k_cache": t["k_cache"][:-1], "v_cache": t["v_cache"][:-1]}


def _gathered(c, t, name):
    """Every sequence's pages one after another, [B, Hkv, S, D] in 32 bits."""
    cache, pages = t[name + "_cache"], t["table"].clamp(min=0).long()
    if c["cache"] == "fp8":
        x = cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * t[name + "_scale"][:, None]
    else:
        x = cache[pages].float()
    return x.flatten(1, 2).transpose(1, 2).contiguous()


def _attention(c, t):
    b, n, hq, dim = t["q"].shape
    group = hq // c["hkv"]
    k, v = _gathered(c, t, "k"), _gathered(c, t, "v")
    q = t["q"].float().view(b, n, c["hkv"], group, dim).permute(0, 2, 3, 1, 4).reshape(b, c["hkv"], group * n, dim)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5
    pos = t["lens"][:, None].long() - n + torch.arange(n, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    s = s.view(b, c["hkv"], group, n, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, c["hkv"], group * n, -1), v).view(b, c["hkv"], group, n, dim)
    o = torch.where(total > 0, o / total, 0.0)
    return {"out": o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, dim).to(t["q"].dtype)}


def _norm(c, t):
    h = t["x"]
    if c["residual"]:
        h = (t["x"].float() + t["r"].float()).to(h.dtype)
    x = h.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * t["w"].float()
    scale = None
    if c["out"] == "fp8":
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / F8_MAX, 1.0)
        y, scale = _in8(y / scale), scale[:, 0]
    else:
        y = y.to(h.dtype)
    return {"y": y, "h": h if c["residual"] else None, "scale": scale}


def _norm_bwd(c, t):
    h, dy, w = t["h"].float(), t["dy"].float(), t["w"].float()
    inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    n = h * inv
    g = dy * w
    dx = inv * (g - n * (g * n).mean(-1, keepdim=True))
    if c["residual"]:
        dx = dx + t["dh"].float()
    return {"dx": dx.to(t["h"].dtype), "dw": (dy * n).sum(0).to(t["w"].dtype)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, e = case, BYTES[case["dtype"]]
    if c["op"] in ("norm", "norm_bwd"):
        n = c["rows"] * c["cols"]
        if c["op"] == "norm_bwd":
            return {"bytes": n * e * (4 if c["residual"] else 3) + 2 * c["cols"] * e, "flops": 12 * n}
        out = BYTES[c["out"]]
        return {"bytes": n * ((3 if c["residual"] else 1) * e + out) + c["cols"] * e + (4 * c["rows"] if out == 1 else 0),
                "flops": (5 if c["residual"] else 4) * n}
    lens, page = _lens(c), c["page"]
    tables = 4 * (len(lens) + sum(-(-n // page) for n in lens))
    rows = c["batch"] * c["new"]
    if c["op"] == "append":
        kept = sum(min(n, c["new"]) for n in lens)
        positions = len({p for n in lens for p in range(max(0, n - c["new"]), n)}) if c["rot"] else 0
        moved = (rows * c["hq"] + kept * (c["hq"] + 2 * c["hkv"])) * c["dim"] * e \
            + kept * 2 * c["hkv"] * c["dim"] * BYTES[c["cache"]]
        return {"bytes": moved + positions * c["rot"] * 4 + 4 * (len(lens) + kept), "flops": 3 * kept * (c["hq"] + c["hkv"]) * c["rot"]}
    read = seen = 0
    for n in lens:
        first = max(0, n - c["new"] + 1 - c["window"]) if c["window"] else 0
        read += n - first
        for t in range(c["new"]):
            last = n - c["new"] + t + 1
            seen += max(0, last - (max(0, last - c["window"]) if c["window"] else 0))
    return {"bytes": 2 * read * c["hkv"] * c["dim"] * BYTES[c["cache"]] + 2 * rows * c["hq"] * c["dim"] * e + tables,
            "flops": 4 * seen * c["hq"] * c["dim"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _e4m3(x):
    """x on the e4m3 grid, nearest, ties to the even step."""
    x = x.clamp(-F8_MAX, F8_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(c, t):
    out = {"q": torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda"),
           "k_cache": t["k_cache"][:-1].double(), "v_cache": t["v_cache"][:-1].double()}
    half = c["rot"] // 2
    for b, n in enumerate(t["lens"].tolist()):
        live = min(n, c["new"])
        if not live:
            continue
        pos = torch.arange(n - live, n, device="cuda")
        got = {name: t[name][b, c["new"] - live:].double() for name in ("q", "k", "v")}
        if half:
            phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                pos.double()[:, None] * _frequencies(c["rot"]).cuda())[:, None]
            re, im = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["pairs"] else (slice(0, half), slice(half, c["rot"]))
            for name in ("q", "k"):
                z = torch.complex(got[name][..., re].contiguous(), got[name][..., im].contiguous()) * phase
                got[name][..., re], got[name][..., im] = z.real, z.imag
        out["q"][b, c["new"] - live:] = got["q"]
        page = t["table"][b].long()[pos // c["page"]]
        for name in ("k", "v"):
            x = got[name]
            if c["cache"] == "fp8":
                x = _e4m3(x / t[name + "_scale"].double()[:, None])
            out[name + "_cache"][page, pos % c["page"]] = x
    return out


def _exact_attention(c, t):
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    group, dim, new = c["hq"] // c["hkv"], c["dim"], c["new"]
    for b, n in enumerate(t["lens"].tolist()):
        if not n:
            continue
        pages = t["table"][b, :-(-n // c["page"])].long()
        k, v = (t[name + "_cache"].view(torch.uint8 if c["cache"] == "fp8" else DTYPES[c["cache"]])[pages].view(
            DTYPES[c["cache"]]).double().flatten(0, 1)[:n] for name in ("k", "v"))
        if c["cache"] == "fp8":
            k, v = k * t["k_scale"].double()[:, None], v * t["v_scale"].double()[:, None]
        for i in range(max(0, new - n), new):
            last = n - new + i + 1
            first = max(0, last - c["window"]) if c["window"] else 0
            ks, vs = k[first:last].transpose(0, 1), v[first:last].transpose(0, 1)
            q = t["q"][b, i].double().view(c["hkv"], group, dim)
            p = torch.softmax(torch.matmul(q, ks.transpose(1, 2).contiguous()) / math.sqrt(dim), -1)
            out[b, i] = torch.matmul(p, vs.contiguous()).view(c["hq"], dim)
    return {"out": out}


def _exact_norm(c, t):
    h = t["x"].double()
    if c["residual"]:
        h = (h + t["r"].double()).to(t["x"].dtype).double()
    y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / c["cols"] + EPS) * t["w"].double()
    scale = None
    if c["out"] == "fp8":
        scale = y.abs().max(-1).values / F8_MAX
        y = _e4m3(y / scale[:, None])
    return {"y": y, "h": h if c["residual"] else None, "scale": scale}


def _exact_norm_bwd(c, t):
    h, dy, w = t["h"].double(), t["dy"].double(), t["w"].double()
    ms = h.square().sum(-1, keepdim=True) / c["cols"] + EPS
    dx = dy * w / ms.sqrt() - h * (dy * w * h).sum(-1, keepdim=True) / (c["cols"] * ms * ms.sqrt())
    if c["residual"]:
        dx = dx + t["dh"].double()
    return {"dx": dx, "dw": (dy * h / ms.sqrt()).sum(0)}


def exact(case, seed):
    t = _inputs(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "norm": _exact_norm,
            "norm_bwd": _exact_norm_bwd}[case["op"]](case, t)
