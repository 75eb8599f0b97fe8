"""Serving operators on the GPU against plain 64-bit implementations: the
product with a packed HiF4 weight, the paged HiF4 cache (append, read) and the
attention over it, and a run of them together.

Tolerances are the roundings counted: one rounding to bf16 is off by at most
2^-8 of the value, a step of an fp32 sum by at most 2^-23 of it (the tensor
cores truncate), summed over the magnitudes that enter.
"""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

L = pytest.importorskip("hif4x._lib")
from hif4x import codec, linalg, serve  # noqa: E402

BF16 = 2.0 ** -8      # half a step of bf16, relative
F32 = 2.0 ** -23      # a whole step of fp32, relative


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def values64(meta, codes):
    """Packed HiF4 (..., nb), (..., nb*32) -> float64 values, element by element from the format."""
    m = meta.cpu().numpy().astype(np.int64) & 0xffffffff
    c = codes.cpu().numpy().reshape(*m.shape, 32)
    nib = np.stack([c & 15, c >> 4], -1).reshape(*m.shape, 64).astype(np.int64)
    e = np.arange(64)
    lv = ((m[..., None] >> (8 + e // 8)) & 1) + ((m[..., None] >> (16 + e // 4)) & 1)
    sf = (1 + (m & 3) / 4) * 2.0 ** (((m & 255) >> 2) - 48)
    v = np.where(nib > 7, -1.0, 1.0) * (nib & 7) / 4 * sf[..., None] * 2.0 ** lv
    return torch.from_numpy(v.reshape(*m.shape[:-1], -1)).cuda()


def packed(seed, *shape, scale=1.0):
    """A packed tensor by the framework's own conversion."""
    x = torch.randn(int(np.prod(shape[:-1])), shape[-1], generator=gen(seed), device="cuda") * scale
    out = codec.convert(x, kind=L.SRC_VALUES, dict5=False, packed=True)
    return out["meta"].view(*shape[:-1], -1), out["codes"].view(*shape[:-1], -1)


def act64(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "gelu":
        return y * 0.5 * (1 + torch.erf(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if act == "silu":
        return y * torch.sigmoid(y)
    return y


def check_linear(x, meta, codes, y, bias=None, act="none", res=None):
    w = values64(meta, codes)
    s = x.double() @ w.t()
    mag = x.double().abs() @ w.abs().t()
    if bias is not None:
        s, mag = s + bias.double(), mag + bias.double().abs()
    z = act64(s, act)
    want = z if res is None else z + res.double()
    # products are exact; C + 8 additions (ranks and bias among them), each at
    # most a step of what is summed; the activations' slopes are below 1.13
    # and their fp32 evaluation within 16 steps of its terms; one rounding
    tol = 1.13 * (x.shape[1] + 8) * F32 * mag + 16 * F32 * (s.abs() + want.abs()) + BF16 * want.abs() * 1.01 + 1e-30
    off = (y.double() - want).abs()
    assert torch.isfinite(y).all()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.2f} of the tolerance"


@pytest.mark.parametrize("T,N,C", [(1, 1, 64), (1, 128, 64), (2, 7, 128), (3, 129, 192), (15, 64, 320), (16, 200, 256),
                                   (17, 130, 448), (33, 256, 1024), (100, 300, 4096), (129, 65, 576), (257, 129, 640),
                                   (300, 1000, 2048), (513, 384, 1088), (1, 4096, 4096), (1, 1000, 14336), (64, 14336, 64)])
def test_linear_sizes(T, N, C):
    meta, codes = packed(T + N + C, N, C, scale=0.02)
    x = torch.randn(T, C, generator=gen(C), device="cuda").bfloat16()
    check_linear(x, meta, codes, serve.linear(x, meta, codes))


@pytest.mark.parametrize("act", list(serve.ACTIVATIONS))
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
def test_linear_epilogue(act, bias):
    T, N, C = 37, 203, 512
    meta, codes = packed(1, N, C, scale=0.1)
    x = torch.randn(T, C, generator=gen(2), device="cuda").bfloat16()
    b = None if bias is None else torch.randn(N, generator=gen(3), device="cuda").to(bias)
    r = torch.randn(T, N, generator=gen(4), device="cuda").bfloat16()
    check_linear(x, meta, codes, serve.linear(x, meta, codes, b, act), b, act)
    check_linear(x, meta, codes, serve.linear(x, meta, codes, b, act, r), b, act, r)


def test_linear_views():
    """Strided x, residual and out; out that is the residual; N and alignments that take no 16-byte stores."""
    T, N, C = 21, 96, 256
    meta, codes = packed(5, N, C)
    wide = torch.randn(T, C + 72, generator=gen(6), device="cuda").bfloat16()
    x = wide[:, 64:64 + C]
    res_wide = torch.randn(T, N + 5, generator=gen(7), device="cuda").bfloat16()
    for cut in (res_wide[:, 5:], res_wide[:, :N], res_wide[:, 1:1 + N]):
        check_linear(x, meta, codes, serve.linear(x, meta, codes, residual=cut), res=cut)
        before = res_wide.clone()
        keep = cut.clone()
        got = serve.linear(x, meta, codes, residual=cut, out=cut)
        assert got.data_ptr() == cut.data_ptr()
        check_linear(x, meta, codes, cut, res=keep)
        cut.copy_(keep)
        assert torch.equal(res_wide, before)      # nothing beside the view was written
    out = torch.full((T, N + 8), 7.0, device="cuda").bfloat16()
    serve.linear(x, meta, codes, out=out[:, :N])
    check_linear(x, meta, codes, out[:, :N])
    assert (out[:, N:] == 7).all()
    one = torch.randn(C, 3, generator=gen(8), device="cuda").bfloat16().t()[:1].contiguous()
    check_linear(one, meta, codes, serve.linear(one, meta, codes))
    assert serve.linear(x[:0], meta, codes).shape == (0, N)


def test_linear_values_of_every_scale():
    """All 256 scale bytes, every lv bit and every code, random: the decode is exact."""
    N, C = 130, 256
    g = gen(9)
    meta = torch.randint(-2 ** 31, 2 ** 31, (N, C // 64), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    meta = (meta & ~255) | (torch.arange(N * (C // 64), device="cuda").view(N, -1) % 200).to(torch.int32)
    codes = torch.randint(0, 256, (N, C // 2), generator=g, device="cuda", dtype=torch.uint8)
    x = torch.zeros(C, C, device="cuda").bfloat16()
    x.fill_diagonal_(1)                                     # each output is one weight
    y = serve.linear(x, meta, codes)
    assert torch.equal(y.double(), values64(meta, codes).t())


def test_linear_special_values():
    meta, codes = packed(10, 64, 128)
    x = torch.zeros(4, 128, device="cuda").bfloat16()
    x[1, 5], x[2, 6] = float("nan"), float("inf")
    y = serve.linear(x, meta, codes)
    assert (y[0] == 0).all() and (y[3] == 0).all() and y[1].isnan().all()
    w = values64(meta, codes)[:, 6]
    assert torch.equal(y[2][w != 0].double(), torch.sign(w[w != 0]) * float("inf"))
    for act in serve.ACTIVATIONS:                            # far arguments stay finite or keep their limit
        x = torch.full((1, 128), 1e4, device="cuda").bfloat16()
        y = serve.linear(x, meta, codes, activation=act)
        check_linear(x, meta, codes, y, act=act)


@pytest.mark.parametrize("T,N,C,runs", [(1, 1000, 14336, 300), (64, 4096, 14336, 100), (300, 1000, 2048, 100),
                                        (2048, 2048, 4096, 30)])
def test_linear_is_reproducible(T, N, C, runs):
    """Every call gives the same bits (a box of codes or a stage reused too early shows here)."""
    meta, codes = packed(31, N, C, scale=0.02)
    x = torch.randn(T, C, generator=gen(C), device="cuda").bfloat16()
    first = serve.linear(x, meta, codes)
    check_linear(x, meta, codes, first)
    same = [torch.equal(serve.linear(x, meta, codes), first) for _ in range(runs)]
    assert all(same), f"{same.count(False)} of {runs} runs differ"


# ------------------------------------------------------------------ the cache
class Batch:
    """A cache with ragged sequences: random pages in random order, `spare` pages that are nobody's."""

    def __init__(self, new, lens, kvh, dh, page, seed, fill=True, spare=3):
        g = np.random.default_rng(seed)
        each = [max(1, -(-n // page)) for n in lens]
        total = sum(each) + spare
        order = g.permutation(total)
        table = np.full((len(lens), max(each) + 1), -7, np.int32)     # entries behind a sequence's pages are no pages
        at = 0
        for i, n in enumerate(each):
            table[i, :n] = order[at:at + n]
            at += n
        self.new, self.lens, self.page, self.kvh, self.dh = new, lens, page, kvh, dh
        self.rows = sum(new)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.pages = torch.tensor(table, device="cuda")
        self.cache = serve.PagedKV.empty(total, page, kvh, dh, "cuda")
        if fill:
            for m, c, s in ((self.cache.k_meta, self.cache.k_codes, 1), (self.cache.v_meta, self.cache.v_codes, 2)):
                pm, pc = packed(seed * 7 + s, total, kvh, page, dh)
                m.copy_(pm)
                c.copy_(pc)

    @property
    def args(self):
        return self.cu, self.len, self.pages

    def values(self, i):
        """(K, V) of sequence i: (kvh, len, dh) float64."""
        out = []
        ids = self.pages[i, :max(1, -(-self.lens[i] // self.page))].long()
        for m, c in ((self.cache.k_meta, self.cache.k_codes), (self.cache.v_meta, self.cache.v_codes)):
            v = values64(m[ids], c[ids]).transpose(0, 1).reshape(self.kvh, -1, self.dh)
            out.append(v[:, :max(0, self.lens[i])])
        return out


SHAPES = [([1], [1], 1, 64, 16), ([1, 1, 1], [5, 17, 300], 2, 128, 16), ([3, 0, 7, 1], [3, 40, 100, 64], 3, 64, 32),
          ([130, 1], [257, 1], 8, 128, 64), ([5] * 70, list(range(5, 75)), 1, 128, 256)]


@pytest.mark.parametrize("new,lens,kvh,dh,page", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_is_the_searched_encode(new, lens, kvh, dh, page, dtype):
    """Every row's bits equal hif4x_convert's, in the right place; nothing else is written; read gives them back."""
    b = Batch(new, lens, kvh, dh, page, 3, fill=False)
    T = b.rows
    x = torch.randn(T + 2, 2, kvh, dh, generator=gen(T), device="cuda")
    x *= torch.exp2(torch.randint(-60, 18, (T + 2, 2, kvh, 1), generator=gen(5), device="cuda").float())
    x[:, 0, :, ::7] = 0
    x[0, 1] = 0
    x = x.to(dtype)
    k, v = x[:, 0], x[:, 1]                                   # strided views; two rows of padding behind
    for t in (b.cache.k_codes, b.cache.v_codes, b.cache.k_meta, b.cache.v_meta):
        t.fill_(77)
    serve.kv_append(b.cache, k, v, *b.args)
    want = {n: torch.full_like(getattr(b.cache, n), 77) for n in ("k_codes", "k_meta", "v_codes", "v_meta")}
    at = 0
    for i, (n, full) in enumerate(zip(new, lens)):
        for j in range(n):
            p = full - n + j
            page_id = int(b.pages[i, p // page])
            for name, src in (("k", k), ("v", v)):
                o = codec.convert(src[at].float().contiguous(), kind=L.SRC_VALUES, dict5=False, packed=True)
                want[name + "_codes"][page_id, :, p % page] = o["codes"]
                want[name + "_meta"][page_id, :, p % page] = o["meta"]
            at += 1
            if at > 150:
                break
        if at > 150:
            break
    if T <= 150:
        for n, w in want.items():
            assert torch.equal(getattr(b.cache, n), w), n
    for dt in (torch.bfloat16, torch.float32):
        rk, rv = (torch.full((T + 2, kvh, dh), 9.0, dtype=dt, device="cuda") for _ in range(2))
        serve.kv_read(b.cache, *b.args, rows=T + 2, out=(rk, rv))
        for got, src in ((rk, k), (rv, v)):
            deq = codec.convert(src[:T].float().reshape(T * kvh, dh).contiguous(), kind=L.SRC_VALUES, dict5=False,
                                deq_dtype=torch.float32)["deq"].view(T, kvh, dh)
            assert torch.equal(got[:T].float(), deq)
            assert (got[T:] == 9).all()
    linalg.check_device_status()


def test_append_unaligned_views():
    b = Batch([9], [30], 2, 64, 16, 4, fill=False)
    for dt in (torch.bfloat16, torch.float32):
        wide = torch.randn(9, 2, 67, generator=gen(1), device="cuda").to(dt)
        k, v = wide[:, :, 1:65], wide[:, :, 3:67]
        serve.kv_append(b.cache, k, v, *b.args)
        gk, gv = serve.kv_read(b.cache, *b.args, rows=9)
        serve.kv_append(b.cache, k.contiguous(), v.contiguous(), *b.args)
        wk, wv = serve.kv_read(b.cache, *b.args, rows=9)
        assert torch.equal(gk, wk) and torch.equal(gv, wv)


def test_places_that_are_none():
    """Rows before position 0 and page entries outside the cache: skipped, reported, nothing else touched."""
    b = Batch([4, 3], [2, 40], 2, 128, 16, 6, fill=False)     # sequence 0: rows 0 and 1 at positions -2 and -1
    x = torch.randn(7, 2, 128, generator=gen(2), device="cuda").bfloat16()
    serve.kv_append(b.cache, x, x, *b.args)
    linalg.check_device_status()
    k, v = (torch.full((7, 2, 128), 3.0, device="cuda").bfloat16() for _ in range(2))
    serve.kv_read(b.cache, *b.args, rows=7, out=(k, v))
    assert (k[:2] == 3).all() and not (k[2:] == 3).all(2).any()
    assert (b.cache.k_meta != 0).any(3).sum() == 5 * 2
    for bad in (-1, b.cache.num_pages, 2 ** 31 - 1):
        keep = [t.clone() for t in (b.cache.k_codes, b.cache.v_codes)]
        table = b.pages.clone()
        table[1, 2] = bad                                      # positions 32 .. 47
        serve.kv_append(b.cache, -x, -x, b.cu, b.len, table)
        with pytest.raises(L.Hif4xError, match="page"):
            linalg.check_device_status()
        own = int(b.pages[1, 2])
        assert torch.equal(b.cache.k_codes[own], keep[0][own]) and torch.equal(b.cache.v_codes[own], keep[1][own])
        linalg.check_device_status()                           # the status was cleared


# ------------------------------------------------------------------ attention
def check_attention(b, q, out, window=0, sinks=0, scale=None):
    g = q.shape[1] // b.kvh
    scale = b.dh ** -0.5 if scale is None else scale
    at = 0
    for i, (n, full) in enumerate(zip(b.new, b.lens)):
        if n == 0:
            continue
        k, v = b.values(i)
        p = torch.arange(full - n, full, device="cuda")[:, None]
        t = torch.arange(max(full, 0), device="cuda")[None]
        see = t <= p
        if window:
            see &= (t > p - window) | (t < sinks)
        for h in range(q.shape[1]):
            qq, kk, vv = q[at:at + n, h].double(), k[h // g], v[h // g]
            s = (qq @ kk.t() * scale).masked_fill(~see, -math.inf)
            w = torch.nan_to_num(torch.softmax(s, 1))          # rows that see nothing: zeros
            want = w @ vv
            got = out[at:at + n, h].double()
            # scores: dh + 4 fp32 steps of the magnitudes; a weight carries that error (and a few steps of
            # exp2 and of its sum) and one rounding to bf16; the result one more
            err = (b.dh + 4) * F32 * abs(scale) * (qq.abs() @ kk.abs().t()).masked_fill(~see, 0).amax(1, keepdim=True) \
                if t.numel() else torch.zeros(n, 1, device="cuda").double()
            # scores are rounded once more in log2 units, relative to their size
            size = s.masked_fill(~see, 0).abs().amax(1, keepdim=True) if t.numel() else err
            rel = 2 * torch.expm1(err + 4 * F32 * size) + BF16 + (full + 64) * F32
            tol = rel * (w @ vv.abs()) * 1.01 + BF16 * want.abs() * 1.01 + 1e-30
            off = (got - want).abs()
            assert (off <= tol).all(), f"sequence {i} head {h}: off by {(off / tol).max().item():.2f} of the tolerance"
        at += n


CASES = [  # new, lens, query heads, kv heads, dh, page
    ([1], [1], 1, 1, 64, 16),
    ([1], [1], 4, 1, 128, 64),
    ([1, 1, 1, 1], [15, 16, 17, 33], 8, 2, 128, 16),
    ([1, 1], [1000, 3], 32, 8, 128, 64),
    ([1], [5000], 16, 2, 64, 256),
    ([1, 1], [700, 129], 16, 1, 128, 32),                     # sixteen query heads to one key head
    ([1], [333], 40, 2, 128, 16),                             # twenty
    ([3, 2, 0, 1], [40, 900, 7, 1], 6, 2, 128, 32),           # three; an empty sequence
    ([2, 5], [2, 77], 10, 2, 64, 16),                         # five; a sequence that begins here
    ([4, 3], [2, 40], 4, 2, 128, 16),                         # rows before position 0 see nothing
    ([17], [17], 8, 8, 128, 16),
    ([128], [128], 4, 4, 128, 64),
    ([129, 1, 40], [129, 64, 1000], 8, 2, 128, 16),
    ([200, 77], [1500, 77], 12, 4, 64, 32),
    ([333], [4000], 8, 1, 128, 128),
    ([64] * 9, [64 * (i + 1) for i in range(9)], 4, 2, 64, 64),
]


@pytest.mark.parametrize("new,lens,qh,kvh,dh,page", CASES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 0), (33, 5), (300, 64), (7, 2000)])
def test_attention(new, lens, qh, kvh, dh, page, window, sinks):
    b = Batch(new, lens, kvh, dh, page, len(new) + qh)
    q = torch.randn(b.rows, qh, dh, generator=gen(b.rows), device="cuda").bfloat16()
    out = serve.paged_attention(q, b.cache, *b.args, window=window, sinks=sinks, max_new=max(new))
    linalg.check_device_status()
    check_attention(b, q, out, window, sinks)
    # max_new only chooses the way there
    for most in (1, None):
        other = serve.paged_attention(q, b.cache, *b.args, window=window, sinks=sinks, max_new=most)
        check_attention(b, q, other, window, sinks)


def test_attention_is_reproducible():
    b = Batch([1] * 5 + [70], [900, 3, 4000, 64, 65, 2000], 2, 128, 64, 1)
    q = torch.randn(b.rows, 8, 128, generator=gen(1), device="cuda").bfloat16()
    for kw in ({}, {"window": 300, "sinks": 70}, {"max_new": 1}):
        first = serve.paged_attention(q, b.cache, *b.args, **kw)
        same = [torch.equal(first, serve.paged_attention(q, b.cache, *b.args, **kw)) for _ in range(200)]
        assert all(same), f"{same.count(False)} runs differ"


@pytest.mark.parametrize("new", [[2, 1], [60, 100]])
def test_attention_views_and_padding(new):
    """q and out as strided views; rows behind the last sequence stay as they were."""
    lens = [70, 300]
    b = Batch(new, lens, 2, 64, 16, 2)
    T = b.rows
    big = torch.randn(T + 3, 3, 8, 64, generator=gen(3), device="cuda").bfloat16()
    q = big[:, 1]
    out = torch.full((8, T + 3, 72), 5.0, device="cuda").bfloat16()
    view = out.transpose(0, 1)[:, :, :64]
    serve.paged_attention(q, b.cache, *b.args, out=view, max_new=max(new))
    check_attention(b, q[:T], view[:T])
    assert (view[T:] == 5).all() and (out[:, :, 64:] == 5).all()


@pytest.mark.parametrize("scale", [-1.0, 0.0, 1e-3, 1.0, 4.0])
@pytest.mark.parametrize("n", [1, 90])
def test_attention_scales_and_peaks(scale, n):
    """Flat to peaked softmax, falling and rising scores (the running reference moves)."""
    b = Batch([n], [2100], 1, 128, 64, 8)
    k = torch.randn(2100, 1, 128, generator=gen(4), device="cuda")
    ramp = torch.linspace(-3, 3, 2100, device="cuda")[:, None, None]
    for sign in (1, -1):
        q = torch.ones(n, 4, 128, device="cuda").bfloat16()
        full = (torch.tensor([0, 2100], dtype=torch.int32, device="cuda"), b.len, b.pages)
        serve.kv_append(b.cache, (0.1 * k + sign * ramp).bfloat16(), k.bfloat16(), *full)
        out = serve.paged_attention(q, b.cache, *b.args, scale=scale, max_new=n)
        check_attention(b, q, out, scale=scale)


def test_attention_special_values():
    """A NaN or infinity in one query row stays in it; what masked places hold does not matter."""
    b = Batch([40], [90], 2, 64, 16, 9)
    q = torch.randn(40, 4, 64, generator=gen(5), device="cuda").bfloat16()
    clean = serve.paged_attention(q, b.cache, *b.args)
    bad = q.clone()
    bad[3, 1, 7], bad[5, 2, 0] = float("nan"), float("inf")
    out = serve.paged_attention(bad, b.cache, *b.args)
    assert out[3, 1].isnan().all() and out[5, 2].isnan().all()
    keep = torch.ones(40, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = keep[5, 2] = False
    assert torch.equal(out[keep], clean[keep])
    # tokens 90 .. 95 of the last page and all other pages: any bytes
    own = set(b.pages[0, :6].tolist())
    for t in (b.cache.k_codes, b.cache.v_codes, b.cache.k_meta, b.cache.v_meta):
        for p in range(b.cache.num_pages):
            if p not in own:
                t[p].fill_(113)
        t[int(b.pages[0, 5]), :, 10:].fill_(255 if t.dtype == torch.uint8 else -1)
    assert torch.equal(serve.paged_attention(q, b.cache, *b.args), clean)


@pytest.mark.parametrize("n", [1, 60])
def test_attention_bad_pages(n):
    """Keys whose page is none count as hidden, and the status tells of it."""
    b = Batch([n], [200], 2, 128, 16, 10)
    q = torch.randn(n, 4, 128, generator=gen(6), device="cuda").bfloat16()
    for bad in (-1, b.cache.num_pages, 2 ** 31 - 1):
        table = b.pages.clone()
        table[0, 3] = bad                                      # tokens 48 .. 63
        out = serve.paged_attention(q, b.cache, b.cu, b.len, table, max_new=n)
        with pytest.raises(L.Hif4xError, match="page"):
            linalg.check_device_status()
        k, v = b.values(0)
        p = torch.arange(200 - n, 200, device="cuda")[:, None]
        t = torch.arange(200, device="cuda")[None]
        hide = (t > p) | ((t >= 48) & (t < 64))
        for h in range(4):
            s = (q[:, h].double() @ k[h // 2].t() / math.sqrt(128)).masked_fill(hide, -math.inf)
            w = torch.softmax(s, 1)
            tol = 3 * BF16 * (w @ v[h // 2].abs())
            assert ((out[:, h].double() - w @ v[h // 2]).abs() <= tol).all()
    # a length that the table has no pages for
    short = b.pages[:, :6]
    serve.paged_attention(q, b.cache, b.cu, b.len, short, max_new=n)
    with pytest.raises(L.Hif4xError, match="page"):
        linalg.check_device_status()


def test_cache_beyond_32_bits():
    """Pages more than 2^32 bytes into the codes, 2^31 into the meta words' bytes and on."""
    pages, kvh, page, dh = 40000, 8, 256, 128
    make = lambda last, dt: torch.empty(pages, kvh, page, last, dtype=dt, device="cuda")  # noqa: E731
    cache = serve.PagedKV(make(64, torch.uint8), make(2, torch.int32), make(64, torch.uint8), make(2, torch.int32))
    assert cache.k_codes.numel() > 2 ** 32
    table = torch.tensor([[39999, 0, 33333], [32768, 39998, 16384]], dtype=torch.int32, device="cuda")
    lens = [700, 520]
    k, v = (torch.randn(sum(lens), kvh, dh, generator=gen(s), device="cuda").bfloat16() for s in (1, 2))
    cu = torch.tensor([0, 700, 1220], dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    serve.kv_append(cache, k, v, cu, ln, table)
    rk, rv = serve.kv_read(cache, cu, ln, table, rows=1220)
    for got, src in ((rk, k), (rv, v)):
        deq = codec.convert(src.float().reshape(-1, dh).contiguous(), kind=L.SRC_VALUES, dict5=False,
                            deq_dtype=torch.float32)["deq"].view(src.shape)
        assert torch.equal(got.float(), deq)
    # the same rows in a small cache give the same attention, for both kernels
    small = serve.PagedKV.empty(6, page, kvh, dh, "cuda")
    near = torch.tensor([[3, 1, 0], [5, 2, 4]], dtype=torch.int32, device="cuda")
    serve.kv_append(small, k, v, cu, ln, near)
    for new in (1, 50):
        q = torch.randn(2 * new, 32, dh, generator=gen(3), device="cuda").bfloat16()
        c = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
        assert torch.equal(serve.paged_attention(q, cache, c, ln, table, max_new=new),
                           serve.paged_attention(q, small, c, ln, near, max_new=new))
    linalg.check_device_status()


# ------------------------------------------------------------------ together
def test_a_layer_of_decoding_in_a_graph():
    """q/k/v products, append, attention and output product with its residual, as a decoding loop runs them: the
    eager steps, and the same steps replayed from one captured graph on another stream, give the same bits."""
    B, H, KV, D, C, page = 3, 8, 2, 64, 512, 16
    wq, wk, wv, wo = (packed(20 + i, n, C, scale=0.05) for i, n in enumerate((H * D, KV * D, KV * D, C)))
    steps = 20
    xs = torch.randn(steps, B, C, generator=gen(11), device="cuda").bfloat16()

    def start():
        b = Batch([1] * B, [0] * B, KV, D, page, 12, fill=False)
        b.pages = torch.arange(B * 4, dtype=torch.int32, device="cuda").view(B, 4)
        b.cache = serve.PagedKV.empty(B * 4, page, KV, D, "cuda")
        b.len = torch.tensor([0, 7, 21], dtype=torch.int32, device="cuda")
        return b

    def layer(b, x):
        b.len += 1
        q = serve.linear(x, *wq).view(B, H, D)
        k = serve.linear(x, *wk).view(B, KV, D)
        v = serve.linear(x, *wv).view(B, KV, D)
        serve.kv_append(b.cache, k, v, *b.args)
        o = serve.paged_attention(q, b.cache, *b.args, window=18, sinks=2, max_new=1)
        return serve.linear(o.view(B, H * D), *wo, residual=x), q, o

    eager = start()
    outs, qs, os_ = zip(*(layer(eager, x) for x in xs))
    linalg.check_device_status()
    for name, w, src, dst in (("q", wq, xs[-1], qs[-1].view(B, -1)),):
        check_linear(src, *w, dst)
    check_linear(os_[-1].view(B, -1), *wo, outs[-1], res=xs[-1])
    eager.lens = eager.len.tolist()
    check_attention(eager, qs[-1], os_[-1], 18, 2)

    b = start()
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(b, x)                                            # warm-up
    torch.cuda.current_stream().wait_stream(side)
    fresh = start()
    b.len.copy_(fresh.len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _, _ = layer(b, x)
    b.len.copy_(fresh.len)
    for i in range(steps):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(y, outs[i]), i


def test_two_graphs_and_two_streams():
    """Calls at once on two streams, and two graphs replayed in turn: each has its own workspace."""
    b = Batch([1, 1], [3000, 2500], 2, 128, 64, 13)
    c = Batch([1], [4000], 2, 128, 64, 14)
    qb = torch.randn(2, 8, 128, generator=gen(1), device="cuda").bfloat16()
    qc = torch.randn(1, 8, 128, generator=gen(2), device="cuda").bfloat16()
    wb, wc = (serve.paged_attention(q, x.cache, *x.args, max_new=1) for q, x in ((qb, b), (qc, c)))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got.append((serve.paged_attention(qb, b.cache, *b.args, max_new=1), wb))
        with torch.cuda.stream(s2):
            got.append((serve.paged_attention(qc, c.cache, *c.args, max_new=1), wc))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = serve.paged_attention(qb, b.cache, *b.args, max_new=1)
    with torch.cuda.graph(g2):
        o2 = serve.paged_attention(qc, c.cache, *c.args, max_new=1)
    for _ in range(3):
        o1.zero_(), o2.zero_()
        g1.replay(), g2.replay()
        assert torch.equal(o1, wb) and torch.equal(o2, wc)


FIRST_CALL = """
import sys; sys.path.insert(0, sys.argv[1])
import torch
from hif4x import serve
x = torch.ones(3, 128, dtype=torch.bfloat16, device="cuda")
meta, codes = torch.full((64, 2), 0xc0, dtype=torch.int32, device="cuda"), torch.full((64, 64), 0x44, dtype=torch.uint8, device="cuda")
cache = serve.PagedKV.empty(4, 16, 1, 64, "cuda")
cu, ln = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 3], [3]))
pages = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
long = torch.randn(60, 4, 64, device="cuda").bfloat16()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = serve.linear(x, meta, codes)
    serve.kv_append(cache, y.view(3, 1, 64), y.view(3, 1, 64), cu, ln, pages)
    o = serve.paged_attention(y.view(3, 1, 64), cache, cu, ln, pages, max_new=3)
    serve.paged_attention(long, cache, cu * 20, ln, pages)
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
assert (y == 128).all() and (o == 128).all(), (y, o)
print("ok")
"""


def test_first_call_of_a_process_in_a_capture():
    """Nothing that a call does the first time only is forbidden while a stream is captured."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hif4-contest_b200")
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, here], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------ refusals
def test_linear_refusals():
    meta, codes = packed(30, 16, 128)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    ok = serve.linear(x, meta, codes)
    bad = [
        (TypeError, (x.float(), meta, codes), {}), (TypeError, (x.half(), meta, codes), {}),
        (TypeError, (x, meta.long(), codes), {}), (ValueError, (x.cpu(), meta, codes), {}),
        (ValueError, (x, meta.cpu(), codes), {}), (ValueError, (x[:, :64], meta, codes), {}),
        (ValueError, (x[:, :96], meta, codes), {}), (ValueError, (x, meta[:8], codes), {}),
        (ValueError, (x, meta, codes[:, ::2]), {}), (ValueError, (x.t(), meta, codes), {}),
        (ValueError, (torch.zeros(4, 132, dtype=torch.bfloat16, device="cuda")[:, 4:], meta, codes), {}),
        (ValueError, (torch.zeros(4, 129, dtype=torch.bfloat16, device="cuda")[:, 1:], meta, codes), {}),
        (ValueError, (x[:1].expand(4, 128), meta, codes), {}), (ValueError, (x[0], meta, codes), {}),
        (ValueError, (x, meta, codes), {"activation": "swish"}),
        (ValueError, (x, meta, codes), {"bias": torch.zeros(15, device="cuda")}),
        (TypeError, (x, meta, codes), {"bias": torch.zeros(16, device="cuda").half()}),
        (ValueError, (x, meta, codes), {"residual": ok[:3]}), (TypeError, (x, meta, codes), {"residual": ok.float()}),
        (ValueError, (x, meta, codes), {"out": x[:, :16]}), (ValueError, (x, meta, codes), {"out": ok[:, :15]}),
        (ValueError, (x, meta[:0], codes[:0]), {}),
    ]
    for err, args, kw in bad:
        with pytest.raises(err):
            serve.linear(*args, **kw)
    wide = torch.zeros(4, 24, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps residual"):
        serve.linear(x, meta, codes, residual=wide[:, :16], out=wide[:, 8:])


def test_cache_refusals():
    b = Batch([2], [20], 2, 64, 16, 15)
    c = b.cache
    with pytest.raises(ValueError):
        serve.PagedKV.empty(4, 24, 2, 64, "cuda")
    with pytest.raises(ValueError):
        serve.PagedKV.empty(4, 16, 2, 96, "cuda")
    with pytest.raises(ValueError):
        serve.PagedKV(c.k_codes, c.k_meta, c.v_codes[:1], c.v_meta)
    with pytest.raises(ValueError):
        serve.PagedKV(c.k_codes[:, :1], c.k_meta[:, :1], c.v_codes[:, :1], c.v_meta[:, :1])   # not contiguous
    with pytest.raises(TypeError):
        serve.PagedKV(c.k_codes, c.k_meta.long(), c.v_codes, c.v_meta)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for k, v, err in ((x, x.float(), TypeError), (x.half(), x.half(), TypeError), (x[:, :1], x[:, :1], ValueError),
                      (x, x[:1], ValueError), (x[..., :32], x[..., :32], ValueError),
                      (x.transpose(1, 2).contiguous().transpose(1, 2), x, ValueError)):
        with pytest.raises(err):
            serve.kv_append(c, k, v, *b.args)
    for args, err in (((b.cu.long(), b.len, b.pages), TypeError), ((b.cu[:1], b.len, b.pages), ValueError),
                      ((b.cu, b.len, b.pages[0]), ValueError), ((b.cu.cpu(), b.len, b.pages), ValueError),
                      ((b.cu, b.len, b.pages[:, :0]), ValueError)):
        with pytest.raises(err):
            serve.kv_append(c, x, x, *args)
        with pytest.raises(err):
            serve.paged_attention(x, c, *args)
    with pytest.raises(TypeError):
        serve.kv_read(c, *b.args, rows=2, dtype=torch.float16)
    with pytest.raises(ValueError):
        serve.kv_read(c, *b.args, rows=3, out=(x, x.clone()))
    with pytest.raises(ValueError):
        serve.kv_read(c, *b.args, rows=2, out=(x, x))


def test_attention_refusals():
    b = Batch([2], [20], 2, 64, 16, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    for args, kw, err in (((q.float(),), {}, TypeError), ((q[:, :3],), {}, ValueError), ((q[:, :, :32],), {}, ValueError),
                          ((q,), {"window": -1}, ValueError), ((q,), {"sinks": 2 ** 31}, ValueError),
                          ((q,), {"max_new": 0}, ValueError), ((q,), {"out": q}, ValueError),
                          ((q,), {"out": q[:1].expand(2, 4, 64)}, ValueError),
                          ((q,), {"out": torch.zeros_like(q)[:1].expand(2, 4, 64)}, ValueError),
                          ((torch.zeros(2, 4, 68, dtype=torch.bfloat16, device="cuda")[:, :, 4:],), {}, ValueError),
                          ((q.cpu(),), {}, ValueError)):
        with pytest.raises(err):
            serve.paged_attention(args[0], b.cache, *b.args, **kw)
    assert serve.paged_attention(q[:0], b.cache, *b.args).shape == (0, 4, 64)
