"""CPU checks of the norm's and the paged cache's entry points: what they
refuse, with which status, before anything reaches a device; and the norm's
backward formula (the GPU tests' oracle) against differences of the forward."""
import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi

lib = _abi.load()


def status(fn, desc):
    st = getattr(lib, fn)(C.byref(desc))
    assert st == _abi.TVK_OK or lib.tvk_last_error()
    return st


def norm(**kw):
    d = _abi.RmsNormDesc()
    d.dtype = d.out_dtype = d.weight_dtype = _abi.TVK_F16
    d.rows, d.cols = 4, 64
    d.x = d.out = d.weight = 16   # never dereferenced by validation
    d.x_stride = d.out_stride = 64
    d.eps = 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"dtype": _abi.TVK_I32}, "UNSUPPORTED"),
    ({"out_dtype": _abi.TVK_F32}, "UNSUPPORTED"), ({"out_dtype": _abi.TVK_F8E5M2}, "UNSUPPORTED"),
    ({"weight_dtype": _abi.TVK_BF16}, "UNSUPPORTED"), ({"out_dtype": _abi.TVK_F8E4M3FN}, "INVALID"),   # no scale
    ({"rows": -1}, "INVALID"), ({"cols": -1}, "INVALID"), ({"eps": -1.0}, "INVALID"), ({"eps": float("nan")}, "INVALID"),
    ({"x": None}, "INVALID"), ({"out": None}, "INVALID"), ({"x_stride": -64}, "INVALID"), ({"out_stride": 63}, "INVALID"),
    ({"residual_out": 16, "residual_out_stride": 0}, "INVALID"), ({"residual": 16, "residual_stride": -1}, "INVALID"),
    ({"rows": 1 << 31}, "UNSUPPORTED"), ({"cols": 1 << 31}, "UNSUPPORTED"), ({"rows": 0, "x": None}, "OK"), ({"cols": 0}, "OK"),
])
def test_norm_refusals(kw, want):
    assert _abi.STATUS_NAMES[status("tvk_rms_norm_fwd", norm(**kw))] == want


def norm_bwd(**kw):
    d = _abi.RmsNormBwdDesc()
    d.dtype = d.weight_dtype = _abi.TVK_BF16
    d.rows, d.cols = 4, 64
    d.dy = d.h = d.dx = d.weight = d.dweight = 16
    d.dy_stride = d.h_stride = d.dx_stride = 64
    d.eps = 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,want", [
    ({"dtype": _abi.TVK_I8}, "UNSUPPORTED"), ({"weight_dtype": _abi.TVK_F16}, "UNSUPPORTED"), ({"rows": -2}, "INVALID"),
    ({"dy": None}, "INVALID"), ({"h": None}, "INVALID"), ({"dx": None}, "INVALID"), ({"dx_stride": 1}, "INVALID"),
    ({"dh": 16, "dh_stride": -64}, "INVALID"), ({"eps": -1e-9}, "INVALID"), ({"cols": 0}, "OK"),
    ({"rows": 0, "dweight": None}, "OK"),
])
def test_norm_bwd_refusals(kw, want):
    assert _abi.STATUS_NAMES[status("tvk_rms_norm_bwd", norm_bwd(**kw))] == want


def test_null_descriptors():
    for fn in ("tvk_rms_norm_fwd", "tvk_rms_norm_bwd", "tvk_paged_append", "tvk_paged_attention"):
        assert getattr(lib, fn)(None) == _abi.TVK_ERR_INVALID
        assert fn.encode() in lib.tvk_last_error()


def cache():
    c = _abi.PagedCache()
    c.dtype = _abi.TVK_F16
    c.pages, c.page_size, c.heads_kv, c.head_dim = 8, 16, 2, 64
    c.k = c.v = c.table = c.seq_lens = 16
    c.k_stride = c.v_stride = _abi.I64x3(16 * 2 * 64, 2 * 64, 64)
    c.table_stride = c.table_width = 4
    return c


def paged(cls, kw):
    d = cls()
    d.cache = cache()
    d.dtype = _abi.TVK_F16
    d.batch, d.new_tokens, d.heads_q = 2, 1, 4
    d.q = 16
    d.q_stride = _abi.I64x3(256, 256, 64)
    if cls is _abi.PagedAppendDesc:
        d.k = d.v = d.q_out = 16
        d.k_stride = d.v_stride = _abi.I64x3(128, 128, 64)
        d.q_out_stride = d.q_stride
    else:
        d.out, d.out_stride, d.scale = 16, d.q_stride, 0.125
    for k, v in kw.items():
        setattr(d.cache if k.startswith("cache_") else d, k.removeprefix("cache_"), v)
    return d


BOTH = [
    ({"dtype": _abi.TVK_F64}, "UNSUPPORTED"), ({"cache_dtype": _abi.TVK_BF16}, "UNSUPPORTED"),
    ({"cache_dtype": _abi.TVK_F8E5M2}, "UNSUPPORTED"), ({"cache_k_scale": 16}, "INVALID"), ({"batch": -1}, "INVALID"),
    ({"new_tokens": -1}, "INVALID"), ({"heads_q": -1}, "INVALID"), ({"cache_pages": -1}, "INVALID"),
    ({"cache_page_size": 0}, "INVALID"), ({"cache_heads_kv": 0}, "INVALID"), ({"cache_head_dim": 0}, "INVALID"),
    ({"cache_table_width": -1}, "INVALID"), ({"cache_table": None}, "INVALID"), ({"cache_seq_lens": None}, "INVALID"),
    ({"cache_k": None}, "INVALID"), ({"cache_v": None}, "INVALID"), ({"q": None}, "INVALID"),
    ({"cache_pages": 1 << 31}, "UNSUPPORTED"), ({"cache_page_size": 1 << 31}, "UNSUPPORTED"),
    ({"cache_k_stride": _abi.I64x3(-1, 1, 1)}, "INVALID"), ({"q_stride": _abi.I64x3(1, -1, 1)}, "INVALID"),
    ({"new_tokens": 1 << 31}, "UNSUPPORTED"), ({"batch": 1 << 30, "new_tokens": 4}, "UNSUPPORTED"), ({"batch": 0}, "OK"),
    ({"new_tokens": 0}, "OK"), ({"cache_head_dim": 2048}, "UNSUPPORTED"), ({"cache_table_stride": -4}, "INVALID"),
]


@pytest.mark.parametrize("kw,want", BOTH + [
    ({"q_out": None}, "INVALID"), ({"k": None}, "INVALID"), ({"rotary": 16, "rotary_dim": 3, "rotary_len": 9}, "INVALID"),
    ({"rotary": 16, "rotary_dim": 66, "rotary_len": 9}, "INVALID"), ({"rotary": 16, "rotary_dim": 0}, "INVALID"),
    ({"rotary": 16, "rotary_dim": 64, "rotary_len": -1}, "INVALID"),
])
def test_append_refusals(kw, want):
    assert _abi.STATUS_NAMES[status("tvk_paged_append", paged(_abi.PagedAppendDesc, kw))] == want


@pytest.mark.parametrize("kw,want", BOTH + [
    ({"out": None}, "INVALID"), ({"heads_q": 3}, "INVALID"), ({"max_len": -1}, "INVALID"), ({"window": -1}, "INVALID"),
    ({"cache_head_dim": 513}, "UNSUPPORTED"), ({"heads_q": 0}, "OK"), ({"out_stride": _abi.I64x3(0, 0, -1)}, "INVALID"),
])
def test_attention_refusals(kw, want):
    assert _abi.STATUS_NAMES[status("tvk_paged_attention", paged(_abi.PagedAttentionDesc, kw))] == want


def test_binding_refuses_other_layouts():
    h = torch.float16
    x, w = torch.zeros((4, 8), dtype=h), torch.zeros(8, dtype=h)
    out8, scale = torch.zeros((4, 8), dtype=torch.float8_e4m3fn), torch.zeros(4)
    make = _abi.make_rms_norm_desc
    make(x, w, x)
    make(x, w, out8, scale=scale)
    for bad in (lambda: make(x, w[:7], x), lambda: make(x, w, out8), lambda: make(x, w, x, scale=scale),
                lambda: make(x, w.double(), x), lambda: make(x, w, x, residual=x[:2]), lambda: make(x.t(), None, x.t()),
                lambda: make(x[0], w, x), lambda: make(x, w, out8, scale=scale[:3]),
                lambda: _abi.make_rms_norm_bwd_desc(x, x, w, x, w.float()),
                lambda: _abi.make_rms_norm_bwd_desc(x.float(), x, w, x, w)):
        with pytest.raises(_abi.TvkError):
            bad()
    k = torch.zeros((3, 16, 2, 8), dtype=h)
    q, kv = torch.zeros((2, 1, 4, 8), dtype=h), torch.zeros((2, 1, 2, 8), dtype=h)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)
    attend, append = _abi.make_paged_attention_desc, _abi.make_paged_append_desc
    attend(q, k, k, q, lens, table)
    append(q, kv, kv, q, k, k, lens, table, rotary=torch.zeros((9, 8)))
    for bad in (lambda: attend(q, k, k[:2], q, lens, table), lambda: attend(q, k, k, q, lens.long(), table),
                lambda: attend(q, k, k, q, lens, table[:1]), lambda: attend(q, k, k, q[:1], lens, table),
                lambda: attend(q.float(), k, k, q, lens, table), lambda: attend(q, k, k, q, lens, table.t()[:2]),
                lambda: attend(q, k.transpose(2, 3), k.transpose(2, 3), q, lens, table),
                lambda: append(q, kv, kv, None, k, k, lens, table), lambda: append(q, kv[:, :, :1], kv, q, k, k, lens, table),
                lambda: append(q, kv, kv, q, k, k, lens, table, rotary=torch.zeros((9, 8), dtype=torch.float64)),
                lambda: attend(q, k, k, q, lens, table, lse=torch.zeros((2, 1, 3)))):
        with pytest.raises(_abi.TvkError):
            bad()


@pytest.mark.parametrize("with_dh", [False, True])
def test_norm_backward_formula_is_the_forwards_derivative(with_dh):
    from tests.test_rms_norm_gpu import oracle_bwd

    g = torch.Generator().manual_seed(0)
    x, w, dy, dh = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 5), (5,), (3, 5), (3, 5)))
    eps = 0.1

    def loss(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
        return (y * dy).sum() + ((x * dh).sum() if with_dh else 0)

    dx, dw, _, _ = oracle_bwd(dy, x, w, dh if with_dh else None, eps)
    step = 1e-5
    for t, grad in ((x, dx), (w, dw)):
        for i in range(t.numel()):
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += step
            down.view(-1)[i] -= step
            diff = (loss(up, w) - loss(down, w)) if t is x else (loss(x, up) - loss(x, down))
            assert abs(diff / (2 * step) - grad.reshape(-1)[i]) < 1e-8


def test_cache_bookkeeping_on_the_host():
    from torchvulkan_amd import decoder

    cache = decoder.PagedKVCache(2, 5, 4, 1, 8, torch.float32, "cpu", max_len=16)
    cache.extend([5, 1])
    assert cache.lens.tolist() == [5, 1] and (cache.table >= 0).sum(1).tolist() == [2, 1]
    for bad in ([1], [-1, 0], [12, 0]):
        with pytest.raises(_abi.TvkError) as e:
            cache.extend(bad)
        assert e.value.status == _abi.TVK_ERR_INVALID
    with pytest.raises(_abi.TvkError) as e:
        cache.extend([8, 4])   # a page more than there are
    assert e.value.status == _abi.TVK_ERR_OOM
    assert cache.lens.tolist() == [5, 1] and (cache.table >= 0).sum() == 3
    cache.release(0)
    cache.extend([0, 15])
    assert cache.lens.tolist() == [0, 16] and sorted(cache.table[1].tolist()) == sorted(set(cache.table[1].tolist()))
    assert (cache.table[0] == -1).all()
    with pytest.raises(_abi.TvkError):
        decoder.PagedKVCache(0, 5, 4, 1, 8)
    x = torch.zeros((2, 4))
    with pytest.raises(_abi.TvkError):
        decoder.rms_norm(x)   # not on a device
    with pytest.raises(_abi.TvkError):
        decoder.rms_norm(x, residual=torch.zeros((2, 5)))
