"""The decoder block's operators as a program uses them: the root-mean-square
norm with its gradients, and a paged key/value cache that prompts and new tokens
are appended to and attended over. Tensors of the vulkan device or of "cuda"; the
calls are queued on the tensors' device's current stream. The reference composes
these operators from element-wise shaders and keeps dense caches."""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import _abi

__all__ = ["rms_norm", "rms_norm_fp8", "rotary_table", "PagedKVCache"]


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


def _check_norm(x, weight, residual) -> None:
    if x.dim() == 0 or (residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype)):
        raise _abi.TvkError(_abi.TVK_ERR_INVALID, "x: [..., cols], and a residual of its shape and dtype, are expected")
    _check_devices(x.device, weight, residual)


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
