"""tvk_paged_append and tvk_paged_attention against the formulas in float64.

Tolerances count roundings, u = 2^-24 being half a float32 step. A rotated
value is two products and a sum in float32 (3 u of their magnitudes) rounded
once to its type (half a step: eps / 2 of the value, 2^-4 and 2^-10 at least in
8 bits). Attention: a score of D products is off by (D + 16) u of their
magnitudes' sum, and its exponential by that and 2 u of the score, twice (the
sum of exponentials has it too); the sums over n keys add n u of the
probability-weighted |v|; a probability rounded to a 16-bit type is off by
eps / 2, and so is the output."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from torchvulkan_amd import _abi

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
F8 = torch.float8_e4m3fn
HALF = torch.float16
BF16 = torch.bfloat16


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def close(got, ref, tol, what):
    got, ref = got.double().cpu(), ref.double()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    over = ((got - ref).abs() - tol).nan_to_num(nan=-1.0)
    assert over.numel() == 0 or over.max() <= 0, f"{what}: {over.max().item():.3e} over the tolerance"


class Cache:
    """A paged cache on the CPU: every slot filled, pages in a random order, lengths as given."""

    def __init__(self, lens, page, hkv, dim, dtype, seed=0, heads_first=False, spare=2, width=None, stale=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.page, self.dim, self.hkv, self.dtype = page, dim, hkv, dtype
        self.pages = sum(need) + spare
        width = max([1, *need]) if width is None else width
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        shape = (self.pages, hkv, page, dim) if heads_first else (self.pages, page, hkv, dim)
        k, v = rand(shape, torch.float32, seed + 1), rand(shape, torch.float32, seed + 2)
        if stale is not None:   # slots that hold no key of a sequence
            mine = torch.zeros((self.pages, page), dtype=torch.bool)
            for b, n in enumerate(lens):
                pos = torch.arange(n)
                mine[self.table[b].long()[pos // page], pos % page] = True
            mine = mine[:, None, :, None] if heads_first else mine[:, :, None, None]
            k, v = torch.where(mine, k, stale), torch.where(mine, v, stale)
        self.k, self.v = k.to(dtype), v.to(dtype)
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.k_scale = self.v_scale = None
        if dtype == F8:
            self.k_scale, self.v_scale = torch.rand(hkv, generator=g) + 0.5, torch.rand(hkv, generator=g) + 0.5

    def values(self, b, n, which):
        """The first n keys or values of sequence b in float64; rows without a page are None's: zeros and a mask."""
        pos = torch.arange(n)
        page = self.table[b].long()[pos // self.page]
        ok = (page >= 0) & (page < self.pages)
        x = (self.k if which == "k" else self.v).double()[page.clamp(0, self.pages - 1), pos % self.page]
        s = self.k_scale if which == "k" else self.v_scale
        return x * s.double()[:, None] if s is not None else x, ok

    def dev(self):
        """(k, v, lens, table), {scales} on the GPU, with the CPU tensors' strides."""
        def there(t):
            out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
            out.view(torch.uint8).copy_(t.view(torch.uint8)) if t.dtype == F8 and t.stride(3) == 1 else out.copy_(t)
            return out

        scales = {} if self.k_scale is None else {"k_scale": self.k_scale.to(DEV), "v_scale": self.v_scale.to(DEV)}
        return (there(self.k), there(self.v), self.lens.to(DEV), self.table.to(DEV)), scales


def attention_oracle(q, cache, scale, window=0, max_len=0):
    """(out, lse, tolerance) in float64."""
    b, new, hq, dim = q.shape
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:3], float("inf"), dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    eps = torch.finfo(q.dtype).eps / 2
    peps = 0 if q.dtype == torch.float32 else eps
    group = hq // cache.hkv
    for i in range(b):
        n = max(0, min(int(cache.lens[i]), cache.table.shape[1] * cache.page))
        n = min(n, max_len) if max_len else n
        if n <= 0:
            continue
        (k, ok), (v, _) = cache.values(i, n, "k"), cache.values(i, n, "v")
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        for t in range(new):
            last = n - new + t + 1
            first = max(0, last - window) if window else 0
            if last <= first:
                continue
            x = q[i, t].double()
            s = torch.einsum("hd,jhd->hj", x, k[first:last]) * scale
            size = torch.einsum("hd,jhd->hj", x.abs(), k[first:last].abs()).nan_to_num(0, 0, 0).amax(-1) * abs(scale)
            s = torch.where(ok[first:last], s, float("-inf"))
            if not ok[first:last].any():
                continue
            p = torch.softmax(s, -1)
            lse[i, t] = torch.logsumexp(s, -1)
            vv = torch.where(ok[first:last, None, None], v[first:last], 0.0)
            out[i, t] = torch.einsum("hj,jhd->hd", p, vv)
            mean = torch.einsum("hj,jhd->hd", p, vv.abs())
            err = (2 * (dim + 16) * size + 4 * s.abs().nan_to_num(0, 0, 0).amax(-1) + 64 + (last - first)) * U
            tol[i, t] = (peps + err[:, None]) * mean + eps * out[i, t].abs() + TINY[q.dtype]
    return out, lse, tol


def check_attention(cache, q, scale=None, window=0, max_len=0, what=""):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    out, lse, tol = attention_oracle(q, cache, scale, window, max_len)
    args, scales = cache.dev()
    qd = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=DEV)
    qd.copy_(q)
    got, got_lse = _abi.paged_attention(qd, *args, max_len=max_len, scale=scale, window=window, **scales)
    torch.cuda.synchronize()
    close(got, out, tol, what)
    finite = lse.isfinite()
    assert torch.equal(got_lse.cpu().isfinite(), finite), what + " lse"
    assert ((got_lse.cpu().double() - lse).abs()[finite] <= 1e-4 * (1 + lse.abs()[finite])).all(), what + " lse"
    again, again_lse = _abi.paged_attention(qd, *args, max_len=max_len, scale=scale, window=window, **scales)
    assert torch.equal(got, again) and torch.equal(got_lse, again_lse), what + ": other bits the second time"
    return got


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300]


@pytest.mark.parametrize("page", [1, 7, 16, 20, 64, 256])
@pytest.mark.parametrize("cache_dtype", ["same", F8])
def test_lengths_and_pages(gpu, page, cache_dtype):
    for dtype in (HALF, BF16):
        cache = Cache(LENS, page, 2, 64, dtype if cache_dtype == "same" else F8, seed=page, heads_first=page % 2 == 1,
                      stale=float("nan"))
        check_attention(cache, rand((len(LENS), 1, 8, 64), dtype, 5), what=f"page {page} {dtype}")


@pytest.mark.parametrize("dim", [1, 8, 16, 32, 40, 48, 64, 80, 96, 112, 128, 160, 192, 256, 264, 512])
@pytest.mark.parametrize("dtype", [HALF, BF16, torch.float32])
def test_dims(gpu, dim, dtype):
    cache = Cache([70, 5, 0, 333], 24, 2, dim, dtype, seed=dim, stale=float("nan"))
    check_attention(cache, rand((4, 1, 6, dim), dtype, 1), what=f"D {dim} {dtype}")
    cache = Cache([70, 5, 0, 333], 24, 2, dim, F8, seed=dim, stale=float("nan"))
    check_attention(cache, rand((4, 2, 6, dim), dtype, 1), what=f"D {dim} {dtype} 8 bits")


# pages of whole 16-key blocks, whose rows are read by other code, in each way of dealing: a wave a sequence, a workgroup, and
# pieces that are joined. What lies around the output's rows is not the call's.
@pytest.mark.parametrize("dim", [1, 16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 224, 256, 264])
@pytest.mark.parametrize("lens,hkv", [([60, 5, 0, 33], 2), ([300, 70, 0, 400], 2), ([3000, 40], 1)])
@pytest.mark.parametrize("dtype", [HALF, BF16, torch.float32])
def test_dims_in_whole_pages(gpu, dim, lens, hkv, dtype):
    for new, cache_dtype in ((1, dtype), (3, dtype), (1, F8)):
        what = f"D {dim} {dtype} {cache_dtype} {lens} {new}"
        cache = Cache(lens, 16, hkv, dim, cache_dtype, seed=dim, stale=float("nan"))
        q = rand((len(lens), new, 3 * hkv, dim), dtype, 1)
        want, _, tol = attention_oracle(q, cache, dim ** -0.5)
        args, scales = cache.dev()
        qd = q.to(DEV)
        around = torch.full((len(lens), new, 3 * hkv + 2, dim + 16), 7.0, dtype=dtype, device=DEV)
        out = around[:, :, 1:-1, 8:8 + dim]
        d = _abi.make_paged_attention_desc(qd, args[0], args[1], out, args[2], args[3],
                                           stream=torch.cuda.current_stream().cuda_stream, **scales)
        _abi.check(_abi.load().tvk_paged_attention(C.byref(d)))
        torch.cuda.synchronize()
        close(out, want, tol, what)
        out.fill_(7.0)
        assert around.eq(7.0).all(), what + ": values around the output's rows were written"


# rows of one key/value head: 1 to several row blocks; tokens in front of a sequence's start see nothing
@pytest.mark.parametrize("hq,hkv,new", [(1, 1, 1), (3, 1, 5), (8, 8, 1), (16, 1, 1), (17, 1, 1), (33, 1, 1), (8, 2, 7),
                                        (4, 2, 16), (64, 2, 2), (6, 3, 40)])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows(gpu, hq, hkv, new, dim):
    cache = Cache([200, 3, 0, 64, 41], 16, hkv, dim, BF16, seed=hq)
    q = rand((5, new, hq, dim), BF16, 3)
    check_attention(cache, q, what=f"{hq}/{hkv} heads, {new} tokens")
    check_attention(cache, q, window=9, what=f"{hq}/{hkv} heads, {new} tokens, window 9")


@pytest.mark.parametrize("window", [1, 31, 32, 33, 100, 511, 5000])
@pytest.mark.parametrize("new", [1, 3])
def test_windows(gpu, window, new):
    cache = Cache([1000, 1, 33, 640, 2001], 20, 2, 64, HALF, seed=window, stale=float("nan"))
    check_attention(cache, rand((5, new, 8, 64), HALF, 2), window=window, what=f"window {window}")


@pytest.mark.parametrize("lens,hkv,dim", [([5000], 1, 128), ([4097, 10, 0, 2222], 2, 64), ([3000, 2999], 4, 80),
                                          ([20011], 2, 128), ([2500], 2, 256)])
@pytest.mark.parametrize("cache_dtype", ["same", F8])
def test_split_keys(gpu, lens, hkv, dim, cache_dtype):
    cache = Cache(lens, 48, hkv, dim, BF16 if cache_dtype == "same" else F8, seed=len(lens), stale=float("nan"))
    check_attention(cache, rand((len(lens), 1, 4 * hkv, dim), BF16, 2), what=f"{lens}")
    check_attention(cache, rand((len(lens), 3, 4 * hkv, dim), BF16, 2), scale=-0.2, what=f"{lens} negative scale")


def test_scales_of_scores(gpu):
    # no scale at all, large scores (one key takes everything) and an infinite one
    cache = Cache([90, 64], 16, 1, 64, HALF, seed=1)
    q = rand((2, 1, 4, 64), HALF, 2)
    check_attention(cache, q, scale=0.0, what="scale 0")
    check_attention(cache, q, scale=30.0, what="scale 30")


@pytest.mark.parametrize("dim", [64, 128, 40])
def test_nan_and_infinite_keys(gpu, dim):
    cache = Cache([90, 64, 50], 16, 1, dim, HALF, seed=1)
    cache.k[cache.table[0, 1], 3] = float("nan")       # a key that is seen: every row of the sequence is NaN
    cache.v[cache.table[1, 2], 5, 0, 7] = float("inf")   # an infinite value: that column is
    q = rand((3, 1, 4, dim), HALF, 2)
    args, _ = cache.dev()
    out, _ = _abi.paged_attention(q.to(DEV), *args)
    out = out.cpu()
    assert out[0].isnan().all()
    assert out[1, 0, :, 7].isinf().all() and out[1, 0, :, :7].isfinite().all()
    assert out[2].isfinite().all()


@pytest.mark.parametrize("dim", [64, 40])
def test_absent_pages(gpu, dim):
    # entries outside the cache are no keys, wherever they stand; lengths outside the table end at it
    cache = Cache([300, 300, 300, 40, 40], 16, 2, dim, HALF, seed=3)
    cache.table[0, 4] = -1
    cache.table[1, 0] = cache.pages
    cache.table[2, :] = 2 ** 31 - 1
    cache.table[3, 1] = -2 ** 31
    cache.lens[1] = 100000
    cache.lens[4] = -5
    check_attention(cache, rand((5, 2, 4, dim), HALF, 1), what="absent pages")


@pytest.mark.parametrize("dim", [64, 40])
def test_max_len(gpu, dim):
    cache = Cache([300, 20, 150], 16, 2, dim, HALF, seed=3)
    check_attention(cache, rand((3, 1, 4, dim), HALF, 1), max_len=150, what="max_len")


@pytest.mark.parametrize("dim", [64, 128, 40])
def test_strides(gpu, dim):
    # queries inside a projection's output, an output in another order, caches inside larger ones, table rows too
    heads = rand((3, 2, 12, dim), BF16, 1).to(DEV)
    q = heads[:, :, :8]
    cache = Cache([100, 7, 260], 16, 2, dim, BF16, seed=4)
    out, _, tol = attention_oracle(q.cpu(), cache, 0.1)
    args, _ = cache.dev()
    both = torch.zeros((cache.pages, 16, 2, 2, dim + 8), dtype=BF16, device=DEV)   # k and v side by side, padded
    both[..., 0, :dim], both[..., 1, :dim] = args[0], args[1]
    k, v = both[..., 0, :dim], both[..., 1, :dim]
    table = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    table[:, 1:1 + args[3].shape[1]] = args[3]
    o = torch.full((8, 3, 2, dim), float("nan"), dtype=BF16, device=DEV).permute(1, 2, 0, 3)
    d = _abi.make_paged_attention_desc(q, k, v, o, args[2], table[:, 1:1 + args[3].shape[1]], scale=0.1,
                                       stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_paged_attention(C.byref(d)))
    close(o, out, tol, "strides")
    # an address that is not a multiple of 16 bytes
    flat = torch.zeros(both.numel() + 1, dtype=BF16, device=DEV)[1:].view(both.shape)
    flat.copy_(both)
    got, _ = _abi.paged_attention(q, flat[..., 0, :dim], flat[..., 1, :dim], args[2], args[3], scale=0.1)
    close(got, out, tol, "unaligned cache")


def test_far_pages(gpu):
    # offsets past 2^32 elements: a cache of 10 GB whose last pages are used
    page, hkv, dim = 64, 8, 128
    pages = (1 << 32) // (page * hkv * dim) + 64
    small = Cache([900, 130], page, hkv, dim, HALF, seed=6, spare=0)
    k, v = (torch.zeros((pages, page, hkv, dim), dtype=HALF, device=DEV) for _ in range(2))
    k[-small.pages:], v[-small.pages:] = small.k.to(DEV), small.v.to(DEV)
    table = torch.where(small.table >= 0, small.table + (pages - small.pages), -1).to(torch.int32).to(DEV)
    q = rand((2, 1, 32, dim), HALF, 2)
    out, _, tol = attention_oracle(q, small, dim ** -0.5)
    got, _ = _abi.paged_attention(q.to(DEV), k, v, small.lens.to(DEV), table)
    close(got, out, tol, "far pages")
    new = rand((2, 1, hkv, dim), HALF, 3).to(DEV)
    _abi.paged_append(None, new, new, k, v, small.lens.to(DEV), table)
    for b, n in enumerate(small.lens.tolist()):
        assert torch.equal(k[table[b, (n - 1) // page], (n - 1) % page], new[b, 0])


def test_streams_and_capture(gpu):
    # one captured step (append, then attention) follows the lengths and the table between its replays
    hkv, dim, page = 2, 128, 16
    cache = Cache([3000, 0, 700], page, hkv, dim, BF16, seed=8, width=256, spare=700)
    args, _ = cache.dev()
    k, v, lens, table = args
    spare = torch.tensor(sorted(set(range(cache.pages)) - set(cache.table.flatten().tolist())), dtype=torch.int32)
    heads = rand((3, 1, 12, dim), BF16, 1).to(DEV)
    q, nk, nv = heads[:, :, :8], heads[:, :, 8:10], heads[:, :, 10:]
    angle = torch.arange(4096, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(0, dim, 2).double() / dim)
    rotary = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)
    qr, out = torch.empty((3, 1, 8, dim), dtype=BF16, device=DEV), torch.empty((3, 1, 8, dim), dtype=BF16, device=DEV)
    lib = _abi.load()

    def step(stream):
        a = _abi.make_paged_append_desc(q, nk, nv, qr, k, v, lens, table, rotary=rotary, stream=stream)
        b = _abi.make_paged_attention_desc(qr, k, v, out, lens, table, stream=stream)
        _abi.check(lib.tvk_paged_append(C.byref(a)))
        _abi.check(lib.tvk_paged_attention(C.byref(b)))

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step(torch.cuda.current_stream().cuda_stream)
    used = 0
    for i in range(5):
        lens += torch.tensor([1, 1, 350 if i == 2 else 1], dtype=torch.int32, device=DEV)
        for b in range(3):
            for at in range(-(-int(lens[b]) // page)):
                if table[b, at] < 0:
                    table[b, at] = spare[used]
                    used += 1
        heads.copy_(rand(heads.shape, BF16, 20 + i))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        captured = out.clone()
        eager, _ = _abi.paged_attention(qr, k, v, lens, table)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            elsewhere, _ = _abi.paged_attention(qr, k, v, lens, table)
        other.synchronize()
        assert torch.equal(captured, eager) and torch.equal(captured, elsewhere), f"replay {i}"
        cache.k, cache.v, cache.lens, cache.table = k.cpu(), v.cpu(), lens.cpu(), table.cpu()
        want, _, tol = attention_oracle(qr.cpu(), cache, dim ** -0.5)
        close(captured, want, tol, f"replay {i}")


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def rotary_table(positions, rot, seed=0):
    angle = torch.rand((positions, rot // 2), generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 100
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def rotated(x, row, interleaved):
    """(x rotated by the table's row, the terms' magnitude) in float64; row None: not rotated."""
    x = x.double()
    size = x.abs()
    if row is None:
        return x, size
    half = row.numel() // 2
    c, s = row[:half].double(), row[half:].double()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, size = x.clone(), size.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def check_append(cache, q, k, v, rotary=None, interleaved=False, what=""):
    args, scales = cache.dev()
    dtype, new, page = k.dtype, k.shape[1], cache.page
    before = args[0].clone(), args[1].clone()
    got = _abi.paged_append(None if q is None else q.to(DEV), k.to(DEV), v.to(DEV), *args,
                            rotary=None if rotary is None else rotary.to(DEV), interleaved=interleaved, **scales)
    torch.cuda.synchronize()
    gk, gv = args[0].float().cpu(), args[1].float().cpu()
    eps = torch.finfo(dtype).eps / 2
    touched = torch.zeros((cache.pages, page), dtype=torch.bool)
    reach = cache.table.shape[1] * page
    for b in range(k.shape[0]):
        n = max(0, min(int(cache.lens[b]), reach))
        for t in range(new):
            pos = n - new + t
            where = int(cache.table[b, pos // page]) if pos >= 0 else -1
            if pos < 0 or not 0 <= where < cache.pages or (rotary is not None and pos >= rotary.shape[0]):
                assert q is None or got[b, t].eq(0).all(), f"{what}: a token without a place"
                continue
            touched[where, pos % page] = True
            row = None if rotary is None else rotary[pos]
            if q is not None:
                y, size = rotated(q[b, t], row, interleaved)
                close(got[b, t], y, eps * y.abs() + (4 * U * size if row is not None else 0) + (TINY[dtype] if row is not None else 0), what + " q")
            for name, x, r, cached in (("k", k, row, gk), ("v", v, None, gv)):
                y, size = rotated(x[b, t], r, interleaved)
                if cache.dtype == F8:
                    s = (cache.k_scale if name == "k" else cache.v_scale).double()[:, None]
                    y = (y / s).clamp(-448, 448)
                    close(cached[where, pos % page], y, 2.0 ** -4 * y.abs() + 2.0 ** -10 + 8 * U * size / s, f"{what} {name}")
                elif r is None:
                    assert torch.equal(cached[where, pos % page], x[b, t].float()), f"{what} {name}"
                else:
                    close(cached[where, pos % page], y, eps * y.abs() + 4 * U * size + TINY[dtype], f"{what} {name}")
    for now, was in ((args[0], before[0]), (args[1], before[1])):
        now, was = now.cpu(), was.cpu()
        size = now.element_size()
        same = (now.contiguous().view(torch.uint8) == was.contiguous().view(torch.uint8)).flatten(2).all(-1)
        assert size and same[~touched].all(), f"{what}: slots of no new token were written"


def tokens(lens, new, hq, hkv, dim, dtype, seed=0):
    x = rand((len(lens), new, hq + 2 * hkv, dim), dtype, seed)
    return x.split([hq, hkv, hkv], 2)


@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 64), (80, 80), (96, 48), (256, 256), (40, 20), (7, 2),
                                     (2, 2), (33, 32), (64, None), (1, None), (1000, 500)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [HALF, BF16, torch.float32])
def test_append_dims(gpu, dim, rot, interleaved, dtype):
    lens = [0, 1, 3, 17, 40]
    table = None if rot is None else rotary_table(50, rot)
    for cache_dtype in (dtype, F8):
        cache = Cache(lens, 16, 2, dim, cache_dtype, seed=dim)
        check_append(cache, *tokens(lens, 3, 4, 2, dim, dtype, 1), rotary=table, interleaved=interleaved,
                     what=f"D {dim} rot {rot} {cache_dtype}")


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("new", [1, 2, 33, 100])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append_pages(gpu, page, new, heads_first):
    lens = [100, 0, 33, 1, 250]
    cache = Cache(lens, page, 3, 64, BF16, seed=page, heads_first=heads_first)
    check_append(cache, *tokens(lens, new, 5, 3, 64, BF16, 1), rotary=rotary_table(260, 64), what=f"page {page} new {new}")
    check_append(cache, None, *tokens(lens, new, 5, 3, 64, BF16, 1)[1:], what="keys and values alone")


def test_append_without_a_place(gpu):
    lens = [100, 100, 100, 90, 30]
    cache = Cache(lens, 16, 2, 64, HALF, seed=2)
    cache.table[0, 6] = -1
    cache.table[1, 5] = cache.pages
    cache.table[2, :] = -2 ** 31
    cache.lens[3] = 1000     # ends at the table's reach, 112
    cache.lens[4] = -7
    check_append(cache, *tokens(lens, 20, 4, 2, 64, HALF, 1), rotary=rotary_table(95, 64), what="no place")


def test_append_saturates(gpu):
    cache = Cache([5], 16, 1, 16, F8, seed=2)
    cache.k_scale[:], cache.v_scale[:] = 0.001, 1.0
    k = torch.full((1, 1, 1, 16), 3.0, dtype=HALF)
    v = torch.zeros((1, 1, 1, 16), dtype=HALF)
    v[..., 0], v[..., 1], v[..., 2], v[..., 3], v[..., 4] = float("inf"), float("-inf"), float("nan"), 500.0, -0.0
    args, scales = cache.dev()
    _abi.paged_append(None, k.to(DEV), v.to(DEV), *args, **scales)
    at = (int(cache.table[0, 0]), 4, 0)
    assert args[0].float().cpu()[at].eq(448).all()
    got = args[1].float().cpu()[at]
    assert got[0] == 448 and got[1] == -448 and got[2].isnan() and got[3] == 448 and got[4] == 0 and got[5:].eq(0).all()


@pytest.mark.parametrize("cache_dtype", [HALF, F8])
def test_append_8bit_codes(gpu, cache_dtype):
    # every float16 value through the 8-bit conversion: the codes torch's conversion gives
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(HALF)
    x = bits.view(1, 256, 2, 128)
    cache = Cache([256], 16, 2, 128, cache_dtype, seed=2)
    cache.k_scale = cache.v_scale = None
    args, _ = cache.dev()
    _abi.paged_append(None, x.to(DEV), x.to(DEV), *args)
    pos = torch.arange(256)
    for c in args[:2]:
        got = c.cpu()[cache.table[0].long()[pos // 16], pos % 16]
        if cache_dtype == HALF:
            assert torch.equal(got.view(torch.int16), x[0].view(torch.int16))
        else:
            f = x[0].float()
            want = torch.where(f.isnan(), f, f.clamp(-448, 448)).to(F8)
            nan = f.isnan()
            assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan]) and got.float()[nan].isnan().all()


@pytest.mark.parametrize("dim,offset", [(64, 0), (64, 1), (40, 0), (128, 4)])
def test_append_in_place_and_strides(gpu, dim, offset):
    # queries rotated over themselves inside the projection's output, at any alignment
    lens = [40, 3]
    cache = Cache(lens, 16, 2, dim, BF16, seed=2)
    args, _ = cache.dev()
    base = rand((2 * 3 * 8 * dim + offset,), BF16, 1)
    heads = base[offset:].view(2, 3, 8, dim)
    q, k, v = heads.split([4, 2, 2], 2)
    table = rotary_table(64, dim)
    dq, dk, dv = base.to(DEV)[offset:].view(2, 3, 8, dim).split([4, 2, 2], 2)
    rd = torch.zeros((64, dim + 3), device=DEV)
    rd[:, 1:1 + dim] = table.to(DEV)
    d = _abi.make_paged_append_desc(dq, dk, dv, dq, *args, rotary=rd[:, 1:1 + dim],
                                    stream=torch.cuda.current_stream().cuda_stream)
    _abi.check(_abi.load().tvk_paged_append(C.byref(d)))
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        for t in range(3):
            row = table[n - 3 + t]
            y, size = rotated(q[b, t], row, False)
            close(dq[b, t], y, 2.0 ** -8 * y.abs() + 4 * U * size + TINY[BF16], "q over itself")
            y, size = rotated(k[b, t], row, False)
            p = n - 3 + t
            at = int(cache.table[b, p // 16]), p % 16
            close(args[0].cpu()[at], y, 2.0 ** -8 * y.abs() + 4 * U * size + TINY[BF16], "k")
            assert torch.equal(args[1].cpu()[at], v[b, t])
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)


# ---------------------------------------------------------------------------
# attention: masked places, how work is dealt
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [32, 64, 80, 128, 256, 40])
@pytest.mark.parametrize("dtype,cache_dtype", [(HALF, HALF), (BF16, BF16), (torch.float32, torch.float32), (BF16, F8)])
def test_masked_places(gpu, dim, dtype, cache_dtype):
    # keys and values that are no numbers where only some of the new tokens see them: the others' rows stay finite
    for lens, window in (([40, 90, 64, 3], 0), ([300, 33, 128, 700], 30), ([4000, 2], 0)):
        cache = Cache(lens, 16, 2, dim, cache_dtype, seed=dim)
        for b, n in enumerate(lens):
            at = lambda p: (cache.table[b, p // 16], p % 16)   # noqa: E731
            cache.v[at(n - 1)][0, 1] = float("nan")
            cache.k[at(n - 2)][1, 0] = float("nan")
            if cache_dtype != F8:
                cache.v[at(n - 1)][1, 3] = float("inf")
                cache.v[at(n - 2)][1, 3] = float("-inf")
                cache.v[at(n - 1)][1, 5] = float("-inf")
            if window and n > window + 4:
                cache.v[at(n - window - 2)][:, 2] = float("nan")   # left behind by the later tokens' windows
        q = rand((len(lens), 4, 12, dim), dtype, 1)
        want, _, tol = attention_oracle(q, cache, dim ** -0.5, window)
        args, scales = cache.dev()
        got, _ = _abi.paged_attention(q.to(DEV), *args, window=window, **scales)
        close(got, want, tol, f"D {dim} {dtype} {cache_dtype} window {window}")
        inf = want.isinf()
        assert torch.equal(got.double().cpu()[inf], want[inf])
        assert got[0, 0].isfinite().all() or window   # its token sees none of them


@pytest.mark.parametrize("lens,hq,hkv,new,dim", [
    ([700 - 9 * i for i in range(70)], 8, 8, 1, 64),                # more segments than run together, whole
    ([1500 - 20 * i for i in range(70)], 8, 4, 1, 64),              # many, in chunks
    ([3000 + i for i in range(40)], 8, 8, 1, 32),                   # many, in stretches
    ([40, 0, 61, 1] * 40, 8, 8, 1, 128), ([128, 100] * 65, 16, 8, 2, 64),   # a wave each
    ([30000] + [5] * 31, 8, 2, 1, 128),                             # one sequence has nearly all the keys
    ([30000] + [5] * 31, 8, 2, 4, 64),
    ([9000, 20], 8, 1, 4, 128), ([5000], 16, 1, 3, 80),             # joined by a second launch
])
@pytest.mark.parametrize("page", [16, 20])
def test_dealing(gpu, lens, hq, hkv, new, dim, page):
    cache = Cache(lens, page, hkv, dim, BF16, seed=len(lens), stale=float("nan"))
    q = rand((len(lens), new, hq, dim), BF16, 3)
    args, _ = cache.dev()
    for max_len in (0, max(lens)):
        got = check_attention(cache, q, max_len=max_len, what=f"{len(lens)} sequences, max_len {max_len}")
        # a captured call joins in a launch of its own, with the same bits
        qd, out = q.to(DEV), torch.empty_like(got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            d = _abi.make_paged_attention_desc(qd, args[0], args[1], out, args[2], args[3], max_len=max_len,
                                               stream=torch.cuda.current_stream().cuda_stream)
            _abi.check(_abi.load().tvk_paged_attention(C.byref(d)))
        for _ in range(3):
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, got)


def test_prompt_chunk(gpu):
    # tokens of a prompt after a cached prefix: many row blocks, each up to its own last key
    cache = Cache([400, 130, 300], 16, 2, 64, BF16, seed=3, stale=float("nan"))
    q = rand((3, 200, 8, 64), BF16, 2)
    check_attention(cache, q, what="prompt")
    check_attention(cache, q, window=50, what="prompt with a window")
