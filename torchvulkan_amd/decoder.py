"""A decoder's operators as a program uses them: the root-mean-square norm and
layer norm with their gradients, both in 8 bits too; products of 8-bit floats with
a scale for each block of 128; a paged key/value cache that prompts and new tokens
are appended to and attended over; the loss against a teacher's top logits with
its gradient; and the drawing of the next token. Tensors of the vulkan device or
of "cuda"; the calls are queued on the tensors' device's current stream. The
reference composes the norms and the loss from element-wise shaders, keeps dense
caches, and has no 8-bit blocks."""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import _abi

__all__ = ["rms_norm", "rms_norm_fp8", "layer_norm", "layer_norm_fp8", "quantize_fp8", "linear_fp8", "distill_loss",
           "sample", "rotary_table", "PagedKVCache"]


def _stream(t: torch.Tensor):
    if t.device.type == "cuda":
        return torch.cuda.current_stream(t.device).cuda_stream
    if t.device.type != "vulkan":
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, f"a tensor on {t.device}: the decoder's operators run on vulkan or cuda devices")
    s = C.c_void_p()
    _abi.check(_abi.load().tvk_get_stream(t.device.index or 0, C.byref(s)))
    return s.value


@functools.lru_cache(maxsize=None)
def _devices() -> int:
    return torch.cuda.device_count()


def _queue(name: str, desc, t: torch.Tensor) -> None:
    """Makes the call with t's device current: its kernels and their scratch are that device's."""
    lib = _abi.load()
    call = getattr(lib, name)
    if _devices() <= 1:
        return _abi.check(call(C.byref(desc)))
    before, device = C.c_int(), t.device.index or 0
    _abi.check(lib.tvk_get_device(C.byref(before)))
    if before.value == device:
        return _abi.check(call(C.byref(desc)))
    _abi.check(lib.tvk_set_device(device))
    try:
        _abi.check(call(C.byref(desc)))
    finally:
        lib.tvk_set_device(before.value)


def _capturing(t: torch.Tensor) -> bool:
    return t.device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class _WithoutGradient(torch.autograd.Function):
    """The results of a call that has no gradient: a backward pass that reaches them ends there with an error, where it
    would go past tensors that know of no inputs."""

    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.name = name
        ctx.set_materialize_grads(False)
        results = tuple(t.detach() for t in tensors[:count])
        return results if count > 1 else results[0]

    @staticmethod
    def backward(ctx, *grads):
        raise _abi.TvkUnsupported(_abi.TVK_ERR_UNSUPPORTED, f"{ctx.name} has no gradient")


def _without_gradient(name: str, results, *inputs):
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in inputs):
        return results
    many = results if isinstance(results, tuple) else (results,)
    return _WithoutGradient.apply(name, len(many), *many, *(t for t in inputs if t is not None))


def _written(t: torch.Tensor) -> None:
    """Autograd learns of a caller's tensor that a kernel wrote."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., cols] as [rows, cols] with contiguous rows (a copy only where the strides allow no view)."""
    t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.shape[-1] <= 1 or t.stride(1) == 1 else t.contiguous()


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        shape, x2 = x.shape, _rows(x)
        r2 = None if residual is None else _rows(residual)
        y = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
        h = x2 if r2 is None else torch.empty(x2.shape, dtype=x.dtype, device=x.device)
        d = _abi.make_rms_norm_desc(x2, weight, y, r2, None if r2 is None else h, None, eps, _stream(x))
        _queue("tvk_rms_norm_fwd", d, x)
        ctx.save_for_backward(h, weight)
        ctx.set_materialize_grads(False)   # no zeros for what nothing was made of
        ctx.eps, ctx.shape, ctx.added = eps, shape, r2 is not None
        if r2 is None:
            return y.view(shape), None
        return y.view(shape), h.view(shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        dy2 = torch.zeros(h.shape, dtype=h.dtype, device=h.device) if dy is None else _rows(dy)
        dh2 = None if dh is None else _rows(dh)
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) \
            if weight is not None and ctx.needs_input_grad[1] else None
        d = _abi.make_rms_norm_bwd_desc(dy2, h, weight, dx, dw, dh2, ctx.eps, _stream(h))
        _queue("tvk_rms_norm_bwd", d, h)
        dx = dx.view(ctx.shape)
        return dx, dw, dx if ctx.added else None, None


def _check_devices(device, *tensors) -> None:
    """Kernels follow every address they are given: none may be another device's, or the host's."""
    for t in tensors:
        if t is not None and t.device != device:
            raise _abi.TvkError(_abi.TVK_ERR_INVALID, f"tensors on {device} and {t.device}")


def _check_norm(x, weight, residual, bias=None) -> None:
    if x.dim() == 0 or (residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype)):
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "x: [..., cols], and a residual of its shape and dtype, are expected")
    _check_devices(x.device, weight, residual, bias)


def rms_norm(x, weight=None, residual=None, eps: float = 1e-5):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension; with a residual (y, h) of h = x + residual
    (tvk_rms_norm_fwd, tvk_rms_norm_bwd). Differentiable in x, weight and residual on the vulkan device; torch's engine
    follows one accelerator's streams, and refuses a backward pass of cuda tensors once the vulkan device is registered."""
    _check_norm(x, weight, residual)
    y, h = _RmsNorm.apply(x, weight, residual, float(eps))
    return y if residual is None else (y, h)


def rms_norm_fp8(x, weight=None, residual=None, eps: float = 1e-5):
    """(y, scale, h): the norm in float8_e4m3fn with a float32 scale for each row, y * scale[..., None] being the norm;
    h is x without a residual. No gradient: a backward pass that reaches the results raises."""
    _check_norm(x, weight, residual)
    x2 = _rows(x.detach())
    y = torch.empty(x2.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
    r2 = None if residual is None else _rows(residual.detach())
    h = None if r2 is None else torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    d = _abi.make_rms_norm_desc(x2, weight, y, r2, h, scale, eps, _stream(x))
    _queue("tvk_rms_norm_fwd", d, x)
    out = y.view(x.shape), scale.view(x.shape[:-1])
    if h is None:
        return *_without_gradient("rms_norm_fp8", out, x, weight), x
    return _without_gradient("rms_norm_fp8", (*out, h.view(x.shape)), x, weight, residual)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        shape, x2 = x.shape, _rows(x)
        r2 = None if residual is None else _rows(residual)
        y = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
        h = x2 if r2 is None else torch.empty(x2.shape, dtype=x.dtype, device=x.device)
        d = _abi.make_layer_norm_desc(x2, weight, bias, y, r2, None if r2 is None else h, None, eps, _stream(x))
        _queue("tvk_layer_norm_fwd", d, x)
        ctx.save_for_backward(h, weight)
        ctx.set_materialize_grads(False)   # no zeros for what nothing was made of
        ctx.eps, ctx.shape, ctx.added, ctx.bias = eps, shape, r2 is not None, None if bias is None else bias.dtype
        if r2 is None:
            return y.view(shape), None
        return y.view(shape), h.view(shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        dy2 = torch.zeros(h.shape, dtype=h.dtype, device=h.device) if dy is None else _rows(dy)
        dh2 = None if dh is None else _rows(dh)
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) \
            if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty(h.shape[1:], dtype=ctx.bias, device=h.device) if ctx.bias and ctx.needs_input_grad[2] else None
        d = _abi.make_layer_norm_bwd_desc(dy2, h, weight, dx, dw, db, dh2, ctx.eps, _stream(h))
        _queue("tvk_layer_norm_bwd", d, h)
        dx = dx.view(ctx.shape)
        return dx, dw, db, dx if ctx.added else None, None


def layer_norm(x, weight=None, bias=None, residual=None, eps: float = 1e-5):
    """(x - mean(x)) / sqrt(var(x) + eps) * weight + bias over the last dimension; with a residual (y, h) of
    h = x + residual (tvk_layer_norm_fwd, tvk_layer_norm_bwd). Differentiable in x, weight, bias and residual where rms_norm
    is. weight and bias have one dtype, x's or float32."""
    _check_norm(x, weight, residual, bias)
    y, h = _LayerNorm.apply(x, weight, bias, residual, float(eps))
    return y if residual is None else (y, h)


def layer_norm_fp8(x, weight=None, bias=None, residual=None, eps: float = 1e-5):
    """(y, scale, h): the norm in float8_e4m3fn with a float32 scale for each 128 columns of a row, scale
    [..., ceil(cols / 128)]; h is x without a residual. No gradient: a backward pass that reaches the results raises."""
    _check_norm(x, weight, residual, bias)
    x2 = _rows(x.detach())
    y = torch.empty(x2.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((x2.shape[0], _abi.blocks_of(x2.shape[1])), dtype=torch.float32, device=x.device)
    r2 = None if residual is None else _rows(residual.detach())
    h = None if r2 is None else torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    d = _abi.make_layer_norm_desc(x2, weight, bias, y, r2, h, scale, eps, _stream(x))
    _queue("tvk_layer_norm_fwd", d, x)
    out = y.view(x.shape), scale.view(*x.shape[:-1], scale.shape[1])
    if h is None:
        return *_without_gradient("layer_norm_fp8", out, x, weight, bias), x
    return _without_gradient("layer_norm_fp8", (*out, h.view(x.shape)), x, weight, bias, residual)


def quantize_fp8(x, block_rows: int = 1):
    """(values, scale): x [..., cols] in float8_e4m3fn with a float32 scale for each 128 columns of a row, scale
    [..., ceil(cols / 128)]; with block_rows 128, for a weight [rows, cols], a scale for each 128 x 128 of it
    (tvk_quantize_f8). No gradient: a backward pass that reaches the results raises."""
    if x.dim() == 0 or (block_rows != 1 and x.dim() != 2):
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "x: [..., cols] is expected, [rows, cols] with blocks of 128 rows")
    x2 = _rows(x.detach())
    out = torch.empty(x2.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((-(-x2.shape[0] // max(1, block_rows)), _abi.blocks_of(x2.shape[1])), dtype=torch.float32, device=x.device)
    _queue("tvk_quantize_f8", _abi.make_quantize_f8_desc(x2, out, scale, block_rows, _stream(x)), x)
    results = (out.view(x.shape), scale if block_rows != 1 else scale.view(*x.shape[:-1], scale.shape[1]))
    return _without_gradient("quantize_fp8", results, x)


def linear_fp8(x, weight, weight_scale, bias=None, x_scale=None, out_dtype=None):
    """x [..., k] times an 8-bit weight [n, k], as quantize_fp8(w, 128) gives it: [..., n] in out_dtype (x's; bfloat16 for an
    8-bit x). x is 8-bit with x_scale [..., ceil(k / 128)], as layer_norm_fp8 gives it, or in 16 or 32 bits, brought
    into that form by the call (tvk_gemm_f8). No gradient: a backward pass that reaches the result raises."""
    if x.dim() == 0 or (x_scale is not None and x_scale.shape[:-1] != x.shape[:-1]):
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "x: [..., k], and x_scale: [..., ceil(k / 128)], are expected")
    _check_devices(x.device, weight, weight_scale, bias, x_scale)
    x2 = _rows(x.detach())
    s2 = None if x_scale is None else x_scale.detach().reshape(x2.shape[0], x_scale.shape[-1])
    out = torch.empty((x2.shape[0], weight.shape[0]), device=x.device,
                      dtype=out_dtype or (torch.bfloat16 if x.dtype == torch.float8_e4m3fn else x.dtype))
    _queue("tvk_gemm_f8", _abi.make_gemm_f8_desc(x2, s2, weight.detach(), weight_scale.detach(), out, bias, _stream(x)), x)
    return _without_gradient("linear_fp8", out.view(*x.shape[:-1], weight.shape[0]), x, weight, weight_scale, bias, x_scale)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, temperature):
        x, i, t = _rows(logits), _rows(index), _rows(teacher)
        loss, softmax, target = (torch.empty(s, dtype=torch.float32, device=x.device) for s in (x.shape[0], (x.shape[0], 2), i.shape))
        d = _abi.make_distill_desc(x, i, t, loss, None, target, temperature, _stream(x), softmax)
        _queue("tvk_distill_fwd", d, x)
        ctx.save_for_backward(x, i, softmax, target)
        ctx.temperature, ctx.shape = temperature, logits.shape
        return loss.view(logits.shape[:-1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, i, softmax, target = ctx.saved_tensors
        dlogits = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d = _abi.make_distill_bwd_desc(x, i, None, target, dloss.reshape(-1), dlogits, ctx.temperature, _stream(x), softmax)
        _queue("tvk_distill_bwd", d, x)
        return dlogits.view(ctx.shape), None, None, None


def distill_loss(logits, index, teacher, temperature: float = 1.0):
    """The loss of every row of logits [..., cols] against a teacher's top logits: index and teacher [..., top], an index
    outside the columns being no entry (tvk_distill_fwd). float32 [...]; differentiable in logits where rms_norm is, the
    teacher's logits being constants."""
    if logits.dim() == 0 or index.shape != teacher.shape or index.dim() != logits.dim() or index.shape[:-1] != logits.shape[:-1]:
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "logits: [..., cols], index and teacher: [..., top] are expected")
    _check_devices(logits.device, index, teacher)
    return _Distill.apply(logits, index, teacher.detach(), float(temperature))


def sample(logits, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob): the next token of every row of logits [..., cols], int64 [...], drawn with the numbers random [...]
    in [0, 1), and the logarithm of the probability that it was drawn with (tvk_sample). temperature, top_k, top_p and min_p
    are numbers, or tensors [...] (float32, top_k int32) of the logits' device that a captured call follows. No gradient: a
    backward pass that reaches the results raises."""
    shape = logits.shape[:-1]
    if logits.dim() == 0 or random.shape != shape:
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "logits: [..., cols] and random: [...] are expected")

    def of_rows(value, dtype, off, name):
        if not isinstance(value, torch.Tensor):
            return None if value == off else torch.full((math.prod(shape),), value, dtype=dtype, device=logits.device)
        if value.shape != shape or value.dtype != dtype:
            raise _abi.TvkError(_abi.TVK_ERR_INVALID, f"{name}: {dtype} {tuple(shape)} is expected, not {value.dtype} {tuple(value.shape)}")
        return value.detach().reshape(-1)

    filters = [of_rows(temperature, torch.float32, 1.0, "temperature"), of_rows(top_k, torch.int32, 0, "top_k"),
               of_rows(top_p, torch.float32, 1.0, "top_p"), of_rows(min_p, torch.float32, 0.0, "min_p")]
    _check_devices(logits.device, random, *filters)
    x = _rows(logits.detach())
    token = torch.empty(x.shape[0], dtype=torch.int64, device=x.device)
    logprob = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    _queue("tvk_sample", _abi.make_sample_desc(x, random.detach().reshape(-1), token, logprob, *filters, _stream(x)), x)
    token, logprob = token.view(shape), logprob.view(shape)
    return token, _without_gradient("sample", logprob, logits, random)


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, device="cpu") -> torch.Tensor:
    """The angles of positions 0 .. positions - 1: float32 [positions, rotary_dim], cosines then sines, from 64 bits.
    append() takes one on its cache's device."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * torch.pow(
        torch.tensor(base, dtype=torch.float64), -torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


class PagedKVCache:
    """Keys and values of up to `batch` sequences in `pages` pages of `page_size` slots, in each of a model's layers: the
    layers share the lengths and the pages' places.

    The host keeps the sequences' lengths and free pages; extend() gives sequences new positions, release() ends one.
    Both only write the device's `table`, `lens` and `new` (how many of each sequence's positions are new), which the calls
    read there, so a captured step (append, attend) replays for other lengths. append and attend have no gradient: a
    backward pass that reaches their results raises. dtype float8_e4m3fn keeps 8 bits, divided by k_scale and v_scale of each head."""

    def __init__(self, batch: int, pages: int, page_size: int, heads_kv: int, head_dim: int, dtype=torch.bfloat16, device="cuda",
                 max_len: int | None = None, layers: int = 1, k_scale=None, v_scale=None):
        if min(batch, pages, page_size, heads_kv, head_dim, layers) <= 0:
            raise _abi.TvkError(_abi.TVK_ERR_INVALID, "PagedKVCache: sizes must be above zero")
        self.page_size, self.max_len = page_size, int(max_len or pages * page_size)
        self.k, self.v = (torch.empty((layers, pages, page_size, heads_kv, head_dim), dtype=dtype, device=device)
                          for _ in range(2))
        self.k_scale, self.v_scale = k_scale, v_scale
        width = -(-self.max_len // page_size)
        self._table = torch.full((batch, width), -1, dtype=torch.int32)
        self._state = torch.zeros((2, batch), dtype=torch.int32)
        self._lens, self._new = self._state[0], self._state[1]
        self._appended, self._captured = False, False
        self._free = list(range(pages - 1, -1, -1))
        self.table, self._device_state = self._table.to(device), self._state.to(device)
        self.lens, self.new = self._device_state[0], self._device_state[1]

    def length(self, b: int) -> int:
        return int(self._lens[b])

    def extend(self, new) -> None:
        """Adds new[b] positions (an int: the same for all) to every sequence, with pages for them; raises and changes
        nothing where a sequence would pass max_len or the pages run out. They are the sequence's new positions until the
        extend() after the next append(), or, once an append() has been captured and may be replayed, until the next."""
        counts = [int(new)] * len(self._lens) if isinstance(new, int) else [int(n) for n in new]
        if len(counts) != len(self._lens) or min(counts) < 0:
            raise _abi.TvkError(_abi.TVK_ERR_INVALID, "extend: a count of at least zero for each sequence is expected")
        lens = self._lens.tolist()
        ends = [n + more for n, more in zip(lens, counts)]
        if max(ends) > self.max_len:
            raise _abi.TvkError(_abi.TVK_ERR_INVALID, f"extend: a sequence of {max(ends)} positions, the cache's longest are {self.max_len}")
        have = [-(-n // self.page_size) for n in lens]
        need = [-(-end // self.page_size) for end in ends]
        if sum(need) - sum(have) > len(self._free):
            raise _abi.TvkOutOfMemory(_abi.TVK_ERR_OOM, f"extend: {sum(need) - sum(have)} pages are wanted, {len(self._free)} are free")
        for b in range(len(ends)):
            for i in range(have[b], need[b]):
                self._table[b, i] = self._free.pop()
        if self._appended or self._captured:
            self._new.zero_()
            self._appended = False
        self._new += torch.tensor(counts, dtype=torch.int32)
        self._lens.copy_(torch.tensor(ends, dtype=torch.int32))
        self._sync(sum(need) != sum(have))

    def release(self, b: int) -> None:
        """Ends sequence b: its pages are free again and its slot of the batch is empty."""
        for i in range(-(-self.length(b) // self.page_size)):
            self._free.append(int(self._table[b, i]))
            self._table[b, i] = -1
        self._lens[b] = self._new[b] = 0
        self._sync(True)

    def _sync(self, table: bool) -> None:
        if table:
            self.table.copy_(self._table)
        self._device_state.copy_(self._state)

    def append(self, q, k, v, rotary=None, interleaved: bool = False, out=None, layer: int = 0):
        """Writes the newest positions' keys and values, rotated as `rotary` says, and returns their rotated queries
        (tokens [batch, new, heads, head_dim]; sequences with fewer new positions are padded in front, and that padding is
        not written and gives zeros). out may be q."""
        _check_devices(self.k.device, q, k, v, rotary, out, self.k_scale, self.v_scale)
        given = out is not None
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None and q is not None else out
        d = _abi.make_paged_append_desc(q, k, v, out, self.k[layer], self.v[layer], self.lens, self.table, rotary, interleaved,
                                        self.k_scale, self.v_scale, _stream(k), self.new)
        _queue("tvk_paged_append", d, k)
        self._appended, self._captured = True, self._captured or _capturing(k)
        if given:
            _written(out)
        return out if out is None else _without_gradient("PagedKVCache.append", out, q, k, v)

    def attend(self, q, scale: float | None = None, window: int = 0, out=None, max_len: int | None = None, layer: int = 0):
        """Attention of the new positions' queries over their sequences (zeros for padding in front of them). max_len: a
        bound on the lengths, past which keys are cut off; without it the longest sequence's, or, in a call that is captured
        and replayed for other lengths, the cache's."""
        _check_devices(self.k.device, q, out, self.k_scale, self.v_scale)
        given = out is not None
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        max_len = max_len or (self.max_len if _capturing(q) else max(1, int(self._lens.max())))
        d = _abi.make_paged_attention_desc(q, self.k[layer], self.v[layer], out, self.lens, self.table,
                                           max_len, scale, window, self.k_scale, self.v_scale, stream=_stream(q),
                                           new_lens=self.new)
        _queue("tvk_paged_attention", d, q)
        if given:
            _written(out)
        return _without_gradient("PagedKVCache.attend", out, q)
