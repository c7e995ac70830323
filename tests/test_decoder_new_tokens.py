"""The paged cache's count of each sequence's new positions, on the host."""
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
