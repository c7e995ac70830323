"""The paged cache of torchvulkan_amd.decoder on the host: the count of each sequence's new positions, and which calls it
makes of the library."""
import pytest
import torch

from torchvulkan_amd import _abi, decoder


@pytest.fixture
def calls(monkeypatch):
    """The calls that would be queued: the entry points themselves are replaced."""
    made = []

    class Library:
        def __getattr__(self, name):
            return lambda d: made.append((name, d._obj)) or 0

    monkeypatch.setattr(_abi, "load", Library)
    monkeypatch.setattr(decoder, "_stream", lambda t: None)
    return made


def test_counts_of_new_positions(calls, monkeypatch):
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, torch.float32, "cpu")
    k = torch.zeros((2, 3, 1, 8))
    cache.extend([3, 1])
    assert cache.new.tolist() == [3, 1]
    cache.extend([0, 1])   # nothing has been appended: these are new too
    assert cache.new.tolist() == [3, 2] and cache.lens.tolist() == [3, 2]
    cache.append(None, k, k)
    cache.append(None, k, k)   # another layer's
    assert calls[-1][1].cache.new_lens == cache.new.data_ptr() and calls[-1][1].cache.seq_lens == cache.lens.data_ptr()
    cache.attend(k)
    assert calls[-1][1].cache.new_lens == cache.new.data_ptr()
    with pytest.raises(_abi.TvkError):
        cache.extend([1000, 0])
    assert cache.new.tolist() == [3, 2]
    cache.extend([1, 0])
    assert cache.new.tolist() == [1, 0] and cache.lens.tolist() == [4, 2]
    cache.release(0)
    assert cache.new.tolist() == [0, 0]
    # a captured append is replayed between extends, unseen by the host
    monkeypatch.setattr(decoder, "_capturing", lambda t: True)
    cache.append(None, k, k)
    monkeypatch.undo()
    for counts in ([1, 1], [1, 0], [0, 1]):
        cache.extend(counts)
        assert cache.new.tolist() == counts


def test_binding_refuses_other_counts():
    h = torch.float16
    k = torch.zeros((3, 16, 2, 8), dtype=h)
    q, kv = torch.zeros((2, 1, 4, 8), dtype=h), torch.zeros((2, 1, 2, 8), dtype=h)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)
    assert _abi.make_paged_attention_desc(q, k, k, q, lens, table, new_lens=lens).cache.new_lens == lens.data_ptr()
    assert _abi.make_paged_append_desc(q, kv, kv, q, k, k, lens, table).cache.new_lens is None
    for bad in (lens[:1], lens.long(), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(_abi.TvkError):
            _abi.make_paged_attention_desc(q, k, k, q, lens, table, new_lens=bad)
        with pytest.raises(_abi.TvkError):
            _abi.make_paged_append_desc(q, kv, kv, q, k, k, lens, table, new_lens=bad)


@pytest.mark.parametrize("other", ["q", "k", "v", "rotary", "out", "k_scale", "v_scale"])
def test_tensors_of_another_device_are_refused(calls, other):
    # "meta" stands for a device that the cache's kernels cannot read
    dtype = torch.float8_e4m3fn if "scale" in other else torch.float32
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, dtype, "cpu", k_scale=torch.ones(1), v_scale=torch.ones(1)) \
        if "scale" in other else decoder.PagedKVCache(2, 40, 4, 1, 8, dtype, "cpu")
    cache.extend(1)
    t = {n: torch.zeros((2, 1, 1, 8)) for n in ("q", "k", "v", "out")}
    t["rotary"] = decoder.rotary_table(9, 8)
    cache.append(**t)
    cache.attend(t["q"], out=t["out"])
    assert len(calls) == 2
    if "scale" in other:
        setattr(cache, other, getattr(cache, other).to("meta"))
    else:
        t[other] = t[other].to("meta")
    with pytest.raises(_abi.TvkError) as e:
        cache.append(**t)
    assert e.value.status == _abi.TVK_ERR_INVALID
    if other not in ("k", "v", "rotary"):
        with pytest.raises(_abi.TvkError):
            cache.attend(t["q"], out=t["out"])
    assert len(calls) == 2


def test_a_captured_call_is_bounded_by_the_cache(calls, monkeypatch):
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, torch.float32, "cpu", max_len=60)
    q = torch.zeros((2, 1, 1, 8))
    cache.extend([7, 3])
    cache.attend(q)
    cache.attend(q, max_len=20)
    monkeypatch.setattr(decoder, "_capturing", lambda t: True)
    cache.attend(q)
    cache.attend(q, max_len=20)
    assert [d.max_len for _, d in calls] == [7, 20, 60, 20]


def test_a_backward_pass_ends_at_calls_without_a_gradient(calls):
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, torch.float32, "cpu")
    x = torch.zeros((2, 1, 1, 8))
    leaf = torch.ones((2, 1, 1, 8), requires_grad=True)
    cache.extend(1)
    for result in (lambda: cache.append(leaf * 2, x, x), lambda: cache.append(x, leaf * 2, x), lambda: cache.append(x, x, leaf * 2),
                   lambda: cache.attend(leaf * 2), lambda: decoder.rms_norm_fp8(leaf * 2)[1],
                   lambda: decoder.rms_norm_fp8(x, residual=leaf * 2)[2],
                   lambda: decoder.rms_norm_fp8(x, leaf.view(-1)[:8])[0].float()):
        with pytest.raises(_abi.TvkUnsupported):
            (result() + leaf.view(-1)[0]).sum().backward()
        with torch.no_grad():
            assert not result().requires_grad
    assert not cache.attend(cache.append(x, x, x)).requires_grad
    assert decoder.rms_norm_fp8(leaf)[2] is leaf
    out = torch.empty_like(x)
    assert cache.attend(x, out=out) is out and cache.append(out, x, x, out=out) is out


def test_a_tensor_that_is_written_is_known_to_autograd(calls):
    # what was kept for a backward pass may not be written behind its back
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, torch.float32, "cpu")
    x = torch.zeros((2, 1, 1, 8))
    cache.extend(1)
    for write in (lambda q: cache.append(q, x, x, out=q), lambda q: cache.attend(x, out=q)):
        q = torch.rand((2, 1, 1, 8))
        w = torch.ones((), requires_grad=True)
        y = q * w
        write(q)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        with torch.inference_mode():
            write(torch.rand((2, 1, 1, 8)))


def test_norm_of_rows_without_values(calls):
    for x in (torch.zeros((3, 5, 0)), torch.zeros((0, 0)), torch.zeros((0, 8)), torch.zeros(0)):
        w = torch.ones(x.shape[-1])
        y, h = decoder.rms_norm(x, w, x)
        assert y.shape == h.shape == x.shape
        y, scale, _ = decoder.rms_norm_fp8(x, w)
        assert y.shape == x.shape and scale.shape == x.shape[:-1]
    assert [(d.rows, d.cols) for _, d in calls[::2]] == [(15, 0), (0, 0), (0, 8), (1, 0)]


@pytest.mark.parametrize("devices,current,want", [(1, 1, []), (2, 0, []), (2, 1, [0, 1])])
def test_calls_are_made_on_their_tensors_device(monkeypatch, devices, current, want):
    made, set_to = [], []

    class Library:
        def tvk_get_device(self, d):
            d._obj.value = set_to[-1] if set_to else current
            return 0

        def tvk_set_device(self, d):
            set_to.append(d)
            return 0

        def __getattr__(self, name):
            return lambda d: made.append((name, set_to[-1] if set_to else current)) or 0

    library = Library()
    monkeypatch.setattr(_abi, "load", lambda: library)
    monkeypatch.setattr(decoder, "_stream", lambda t: None)
    monkeypatch.setattr(decoder, "_devices", lambda: devices)
    cache = decoder.PagedKVCache(2, 40, 4, 1, 8, torch.float32, "cpu")
    x = torch.zeros((2, 1, 1, 8))
    cache.extend(1)
    for name, call in (("tvk_paged_append", lambda: cache.append(x, x, x)), ("tvk_paged_attention", lambda: cache.attend(x)),
                       ("tvk_rms_norm_fwd", lambda: decoder.rms_norm(x)), ("tvk_rms_norm_fwd", lambda: decoder.rms_norm_fp8(x))):
        made.clear()
        set_to.clear()
        call()
        assert made == [(name, 0 if devices > 1 else current)] and set_to == want
