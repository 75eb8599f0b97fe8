"""Serving operators on the GPU at the edges of their contract: what a batch may hold that its tensors do not, page
tables with entries that are none, the device status, far arguments of the activations, tensors that overlap, mixed
batches.  Tolerances count roundings as in test_serve_gpu.py."""
import copy
import math

import numpy as np
import pytest
import torch

from test_serve_gpu import BF16, Batch, check_attention, check_linear, gen, packed, values64

pytestmark = pytest.mark.gpu

L = pytest.importorskip("hif4x._lib")
from hif4x import codec, linalg, serve  # noqa: E402


# ------------------------------------------------------------------ values that are none
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_values_that_are_none(dtype):
    """NaN, infinities, the type's largest and smallest values: the bits are hif4x_convert's, and other rows' too."""
    T, kvh, dh = 40, 2, 128
    b = Batch([T], [T], kvh, dh, 16, 56, fill=False)
    x = torch.randn(2, T, kvh, dh, generator=gen(57), device="cuda")
    nan, inf, fi = float("nan"), float("inf"), torch.finfo(dtype)
    specials = (nan, inf, -inf, fi.max, -fi.max, fi.tiny, -fi.tiny, fi.smallest_normal / 8, 0.0, -0.0)
    for i, value in enumerate(specials):
        x[0, i, 0, 5] = value                                    # one in a group
        x[0, 10 + i, 1, 64:] = value                             # a group of them
        x[1, 20 + i, 0, ::3] = value                             # many among others
        x[1, 20 + i, 0, 1] = specials[i - 1]
    for i, size in enumerate((0.0, 2.0 ** -60, 2.0 ** 30)):      # NaN among values whose scales meet the E6M2 limits
        x[0, 30 + i] *= size
        x[0, 30 + i, :, 3:40:9] = nan
    x = x.to(dtype)
    serve.kv_append(b.cache, x[0], x[1], *b.args)
    for src, meta, codes in ((x[0], b.cache.k_meta, b.cache.k_codes), (x[1], b.cache.v_meta, b.cache.v_codes)):
        want = codec.convert(src.float().reshape(T * kvh, dh).contiguous(), kind=L.SRC_VALUES, dict5=False, packed=True)
        at = torch.arange(T, device="cuda")
        ids = b.pages[0].long()[at // 16]
        assert torch.equal(meta[ids, :, at % 16].reshape(T * kvh, -1), want["meta"])
        assert torch.equal(codes[ids, :, at % 16].reshape(T * kvh, -1), want["codes"])
    linalg.check_device_status()


# ------------------------------------------------------------------ rows that the tensors do not have
def cut(b, rows):
    """The batch of b's first `rows` rows: later rows and the keys only they see are gone."""
    c, left = copy.copy(b), rows
    c.new, c.lens = [], []
    for n, full in zip(b.new, b.lens):
        have = min(n, left)
        left -= have
        c.new.append(have)
        c.lens.append(full - n + have)
    return c


@pytest.mark.parametrize("new,lens,qh,kvh,dh,rows", [
    ([40, 60], [100, 200], 4, 2, 64, 70),               # the last sequence is cut
    ([300, 300], [2000, 5000], 8, 2, 128, 200),         # and the one after it has no rows at all
    ([300], [700], 4, 1, 64, 100),                      # most of a sequence is cut
    ([2000, 60], [2000, 200], 8, 2, 128, 100),
    ([300], [9000], 4, 1, 128, 100),                    # with the keys in shares
    ([64, 64], [9000, 9000], 4, 1, 128, 70),
    ([1, 64, 100, 2], [700, 64, 3000, 9], 8, 4, 64, 90),
    ([20] * 8, list(range(40, 840, 100)), 8, 1, 64, 50),
    ([1, 1, 1], [900, 33, 5000], 4, 2, 128, 2)])        # single tokens
def test_rows_the_tensors_do_not_have(new, lens, qh, kvh, dh, rows):
    """A batch description that goes on behind the rows of q: the rows that q has come out right, whatever
    kernel takes them."""
    b = Batch(new, lens, kvh, dh, 16, 41)
    q = torch.randn(rows, qh, dh, generator=gen(rows), device="cuda").bfloat16()
    c = cut(b, rows)
    for most in (max(new), None, 1):
        out = torch.full_like(q, float("nan"))
        serve.paged_attention(q, b.cache, *b.args, max_new=most, out=out)
        linalg.check_device_status()
        check_attention(c, q, out)


# ------------------------------------------------------------------ pages that no row sees
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("new,lens,qh,kvh,dh", [([1, 2], [3000, 700], 4, 2, 128),            # few rows
                                                ([60, 200], [3000, 1531], 4, 2, 128),        # tiles
                                                ([300, 1], [2047, 1999], 8, 8, 64),          # both
                                                ([70], [5000], 4, 1, 128)])                  # keys in shares
@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 4), (1024, 20), (1, 130), (333, 1)])
def test_pages_that_no_row_sees_may_be_none(new, lens, qh, kvh, dh, page, window, sinks):
    """Table entries of pages that hold no visible key (those outside the window and the sinks, given back) may name
    no page: the result is right and nothing is reported."""
    b = Batch(new, lens, kvh, dh, page, 42)
    q = torch.randn(b.rows, qh, dh, generator=gen(window), device="cuda").bfloat16()
    table = b.pages.clone()
    freed = 0
    for i, (n, full) in enumerate(zip(new, lens)):
        p, t = np.arange(full - n, full)[:, None], np.arange(full)[None]
        seen = ((t <= p) & ((t > p - window) | (t < sinks))).any(0)
        for j in range(-(-full // page)):
            if not seen[j * page:(j + 1) * page].any():
                table[i, j] = -1
                freed += 1
    assert freed > 0
    for most in (max(new), None):
        out = serve.paged_attention(q, b.cache, b.cu, b.len, table, window=window, sinks=sinks, max_new=most)
        linalg.check_device_status()
        check_attention(b, q, out, window, sinks)


# ------------------------------------------------------------------ the device status
def bad_page():
    """One append whose page is none."""
    cache = serve.PagedKV.empty(2, 16, 1, 64, "cuda")
    x = torch.ones(1, 1, 64, device="cuda").bfloat16()
    cu, one, table = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [1], [[5]]))
    serve.kv_append(cache, x, x, cu, one, table)


def test_a_bad_page_is_not_the_conversions_affair():
    """A conversion on the same device neither fails for a serving call's bad page nor takes its report."""
    from hif4x import linear, synth
    pair = synth.nvfp4_pair(synth.codec_c1(3, 8, 128))
    linalg.check_device_status()
    bad_page()
    linear.dynamic_activation(*pair, None)
    with pytest.raises(L.Hif4xError, match="page"):
        linalg.check_device_status()
    linalg.check_device_status()


@pytest.mark.parametrize("first", ["wait", "page"])
def test_a_bad_page_does_not_hide_an_expired_wait(first):
    """Both are reported, the expired wait (whose results are void) first, whichever came first."""
    status = lambda: L.lib().hif4x_device_status(L.stream())  # noqa: E731
    done = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert status() == L.OK
    wait = lambda: L.lib().hif4x_wait_selftest(1000, L.ptr(done), L.stream())  # noqa: E731
    for event in (wait, bad_page) if first == "wait" else (bad_page, wait):
        event()
    assert [status() for _ in range(3)] == [L.TIMEOUT, L.BAD_PAGE, L.OK]


def test_a_conversion_still_learns_of_an_expired_wait():
    from hif4x import linear, synth
    done = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert L.lib().hif4x_wait_selftest(1000, L.ptr(done), L.stream()) == L.OK
    with pytest.raises(L.Hif4xError):
        linear.dynamic_activation(*synth.nvfp4_pair(synth.codec_c1(3, 8, 128)), None)
    linalg.check_device_status()


# ------------------------------------------------------------------ far arguments of the activations
def activation_of(v, act):
    """act(v) by serve.linear: a weight of zeros and the bias v, so nothing is rounded before the activation."""
    n = v.numel()
    x = torch.ones(1, 64, device="cuda").bfloat16()
    meta, codes = torch.zeros(n, 1, dtype=torch.int32, device="cuda"), torch.zeros(n, 32, dtype=torch.uint8, device="cuda")
    return serve.linear(x, meta, codes, bias=v, activation=act)[0].double()


def test_gelu_tanh_of_negative_arguments():
    """One rounding to bf16 is all that a value far left of zero loses.  2z carries up to eight fp32 half steps, which the exponential
    turns into 2|z| times as many of its own; exp, sum and quotient add a few."""
    v = torch.cat((torch.linspace(-9, 0, 4001), torch.linspace(0, 12, 501))).cuda()
    z = math.sqrt(2 / math.pi) * (v.double() + 0.044715 * v.double() ** 3)
    want = v.double() * torch.sigmoid(2 * z)
    tol = want.abs() * (BF16 * 1.01 + (8 * 2 * z.abs() + 16) * 2.0 ** -24)
    off = (activation_of(v, "gelu_tanh") - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol.clamp_min(1e-300)).max().item():.2f} of the tolerance"


def test_silu_of_far_negative_arguments():
    """Down to where bf16 has no value left (half its last step is 2^-134), the result is the formula's: exp(-v) passes
    fp32's range at v = -88.7, the result bf16's smallest normal value only behind it."""
    v = torch.cat((torch.linspace(-110, -80, 6001), torch.linspace(-80, 110, 1901))).cuda()
    want = v.double() * torch.sigmoid(v.double())
    # exp within two steps of fp32 (2^-149 each where it has no more bits), product and quotient half a step each
    tol = want.abs() * (BF16 * 1.01 + 16 * 2.0 ** -24) + 1.01 * 2.0 ** -134 + 4 * v.double().abs() * 2.0 ** -149
    off = (activation_of(v, "silu") - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.2f} of the tolerance"


# ------------------------------------------------------------------ tensors that overlap, and what is refused
def test_out_overlaps_no_input():
    """`out` may lie over no tensor that the call reads (in linear the residual itself excepted)."""
    T, N, C = 4, 64, 128
    meta, codes = packed(50, N, C)
    x = torch.zeros(T, C, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps bias"):
        serve.linear(x, meta, codes, bias=flat[:N], out=flat[:T * N].view(T, N))
    with pytest.raises(ValueError, match="overlaps codes"):
        serve.linear(x, meta, flat.view(torch.uint8)[:N * C // 2].view(N, C // 2), out=flat[:T * N].view(T, N))
    with pytest.raises(ValueError, match="overlaps meta"):
        serve.linear(x, flat.view(torch.int32)[:N * C // 64].view(N, C // 64), codes, out=flat[:T * N].view(T, N))
    b = Batch([2], [20], 2, 64, 16, 51)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    c = b.cache
    for t in (c.k_codes, c.k_meta, c.v_codes, c.v_meta):
        over = t.view(-1).view(torch.bfloat16)
        if over.numel() < 512:
            continue
        with pytest.raises(ValueError, match="overlaps the cache"):
            serve.paged_attention(q, c, *b.args, out=over[:512].view(2, 4, 64))
        with pytest.raises(ValueError, match="overlaps the cache"):
            serve.kv_read(c, *b.args, rows=2, out=(over[:256].view(2, 2, 64), torch.zeros(2, 2, 64, device="cuda").bfloat16()))
    table = torch.zeros(1, 256, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlaps pages"):
        serve.paged_attention(q, c, b.cu, b.len, table, out=table.view(torch.bfloat16).view(2, 4, 64))


@pytest.mark.parametrize("T", [1, 5, 300])
def test_out_beside_an_input_in_one_buffer(T):
    """Two column ranges of one buffer never meet: x and out, residual and out, q and out may lie so."""
    N, C = 96, 128
    meta, codes = packed(52, N, C)
    wide = torch.randn(T, C + 2 * N, generator=gen(T), device="cuda").bfloat16()
    x, res, out = wide[:, :C], wide[:, C:C + N], wide[:, C + N:]
    keep = wide.clone()
    serve.linear(x, meta, codes, residual=res, out=out)
    check_linear(x, meta, codes, out, res=res)
    assert torch.equal(wide[:, :C + N], keep[:, :C + N])
    b = Batch([T], [T + 40], 2, 64, 16, 53)
    both = torch.randn(T, 2, 4, 64, generator=gen(T + 1), device="cuda").bfloat16()
    q = both[:, 0].clone()
    serve.paged_attention(both[:, 0], b.cache, *b.args, out=both[:, 1])
    check_attention(b, q, both[:, 1])
    assert torch.equal(both[:, 0], q)
    # and ranges that do meet are refused
    if T > 1:
        with pytest.raises(ValueError, match="overlaps x"):
            serve.linear(x, meta, codes, out=wide[:, C - 8:C - 8 + N])


def test_the_cache_keeps_its_tensors():
    """A cache describes the tensors it was made with: they and its sizes cannot be replaced."""
    c = serve.PagedKV.empty(2, 16, 1, 64, "cuda")
    for name in ("k_codes", "k_meta", "v_codes", "v_meta", "num_pages", "kv_heads", "page_size", "head_dim"):
        with pytest.raises(AttributeError, match=name):
            setattr(c, name, getattr(c, name))


def test_inputs_that_require_a_gradient():
    """There is no backward pass, so such inputs are refused where gradients are recorded and taken elsewhere."""
    meta, codes = packed(54, 64, 128)
    x = torch.randn(2, 128, generator=gen(1), device="cuda").bfloat16()
    r, bias = torch.zeros(2, 64, device="cuda").bfloat16(), torch.zeros(64, device="cuda")
    g = lambda t: t.clone().requires_grad_()  # noqa: E731
    b = Batch([2], [20], 1, 64, 16, 55)
    kv, q = torch.zeros(2, 1, 64, device="cuda").bfloat16(), torch.zeros(2, 1, 64, device="cuda").bfloat16()
    calls = [lambda: serve.linear(g(x), meta, codes), lambda: serve.linear(x, meta, codes, bias=g(bias)),
             lambda: serve.linear(x, meta, codes, residual=g(r)), lambda: serve.linear(x, meta, codes, out=g(r)),
             lambda: serve.kv_append(b.cache, g(kv), kv, *b.args), lambda: serve.kv_append(b.cache, kv, g(kv), *b.args),
             lambda: serve.kv_read(b.cache, *b.args, rows=2, out=(g(kv), kv.clone())),
             lambda: serve.paged_attention(g(q), b.cache, *b.args),
             lambda: serve.paged_attention(q, b.cache, *b.args, out=g(q))]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    assert not serve.linear(x, meta, codes).requires_grad


# ------------------------------------------------------------------ batches of both kinds
def work_bytes(page, kvh, dh, B, most, qh, rows, max_new, window=0, sinks=0):
    need = L.i64()
    L.call("hif4x_paged_attention_work", page, kvh, dh, B, most, qh, rows, window, sinks, max_new, need)
    return need.value


def test_single_tokens_beside_a_chunk_share_their_keys():
    """A long token beside a chunk, and a decoding batch whose call does not say max_new: the keys of the single tokens are shared out
    as they are in a call of their own (the workspace holds a sum for each share, and is bounded)."""
    slot = 16 * (128 + 2) * 4                                   # sums of a key head's rows of one share, in bytes
    mixed = work_bytes(64, 8, 128, 2, 1024, 32, 2049, 2048)
    assert mixed >= 16 * 2 * 8 * slot, mixed
    unsaid = work_bytes(64, 8, 128, 64, 128, 32, 64, 64)
    assert unsaid >= 3 * 64 * 8 * slot, unsaid
    assert max(mixed, unsaid) <= 2 ** 29 + 2 ** 24
    assert work_bytes(64, 8, 128, 2, 7, 32, 300, 299) == 0      # short contexts: one launch of each kernel


@pytest.mark.parametrize("new,lens,qh,kvh,dh,page", [
    ([1, 200], [20000, 900], 8, 2, 128, 64), ([200, 1], [900, 20000], 8, 2, 128, 64),
    ([64, 1, 64, 2], [9000, 9000, 300, 7000], 4, 1, 64, 16),     # both kinds in shares
    ([1] * 9 + [0, 40], [5000 + i for i in range(9)] + [3, 40], 8, 4, 128, 32),
    ([17, 16, 1, 15], [6000, 6000, 6000, 6000], 1, 1, 64, 16),   # about the border of the two kernels
    ([5, 6, 5], [6000, 3000, 2], 3, 1, 128, 16)])                # three query heads; rows that see nothing
@pytest.mark.parametrize("window,sinks", [(0, 0), (2500, 3)])
def test_batches_of_both_kinds(new, lens, qh, kvh, dh, page, window, sinks):
    b = Batch(new, lens, kvh, dh, page, 43)
    q = torch.randn(b.rows + 3, qh, dh, generator=gen(7), device="cuda").bfloat16()
    first = None
    for _ in range(5):
        out = torch.full_like(q, 5.0)
        serve.paged_attention(q, b.cache, *b.args, window=window, sinks=sinks, out=out)
        assert (out[b.rows:] == 5).all()                         # padding rows stay as they were
        first = out if first is None else first
        assert torch.equal(out, first)
    linalg.check_device_status()
    check_attention(b, q, first, window, sinks)


# ------------------------------------------------------------------ every scale byte, level bit and code
def every_byte(shape, seed):
    """Packed units (shape) x 64 elements with random levels and codes, the scale bytes 0 .. 255 in turn."""
    g = gen(seed)
    n = math.prod(shape)
    meta = torch.randint(-2 ** 23, 2 ** 23, (n,), generator=g, device="cuda") << 8 | torch.arange(n, device="cuda") % 256
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] * 32), generator=g, device="cuda", dtype=torch.uint8)
    return meta.to(torch.int32).view(shape), codes


def test_linear_of_every_scale_byte():
    meta, codes = every_byte((130, 4), 60)
    x = torch.eye(256, device="cuda").bfloat16()                 # each output is one weight
    assert torch.equal(serve.linear(x, meta, codes).double(), values64(meta, codes).t())


@pytest.mark.parametrize("dh", [64, 128])
def test_cache_of_every_scale_byte(dh):
    """kv_read, and V in both attention kernels (a window of one key: the result is that key's V)."""
    pages, kvh, page = 24, 2, 16
    shape = (pages, kvh, page, dh // 64)
    (km, kc), (vm, vc) = every_byte(shape, 61), every_byte(shape, 62)
    cache = serve.PagedKV(kc, km, vc, vm)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    n = pages * page
    order = lambda m, c: values64(m, c)[table[0].long()].transpose(1, 2).reshape(n, kvh, dh)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = serve.kv_read(cache, i32(0, n), i32(n), table, rows=n)
    assert torch.equal(k.double(), order(km, kc)) and torch.equal(v.double(), order(vm, vc))
    q = torch.zeros(n, 4, dh, device="cuda").bfloat16()
    out = serve.paged_attention(q, cache, i32(0, n), i32(n), table, window=1)
    assert torch.equal(out.double(), order(vm, vc).repeat_interleave(2, 1))
    # a row a sequence, each with its own length
    cu, lens = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.arange(1, n + 1, dtype=torch.int32, device="cuda")
    out = serve.paged_attention(q, cache, cu, lens, table.expand(n, pages).contiguous(), window=1, max_new=1)
    assert torch.equal(out.double(), order(vm, vc).repeat_interleave(2, 1))
    linalg.check_device_status()


@pytest.mark.parametrize("n", [1, 17])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_with_keys_of_every_scale_byte(n, dh):
    """K in both attention kernels: sequence s has the scale byte s in all its keys and queries of that much less size."""
    b = Batch([n] * 256, [n + 9] * 256, 1, dh, 32, 63)
    E = torch.arange(256, device="cuda") // 4 - 48
    for s in range(256):
        ids = b.pages[s, :1].long()
        b.cache.k_meta[ids] = (b.cache.k_meta[ids] & ~255) | s
    q = torch.randn(256, n, 1, dh, generator=gen(64), device="cuda") * torch.exp2(-E.float())[:, None, None, None]
    q = q.reshape(256 * n, 1, dh).bfloat16()
    check_attention(b, q, serve.paged_attention(q, b.cache, *b.args, max_new=n))


# ------------------------------------------------------------------ weights of another space
def to_weight_space(x, s, mode):
    """x as the product with a calibrated weight takes it: smoothed and, by mode, rotated."""
    return codec.convert(x, kind=L.SRC_VALUES, smooth=s, smooth_mode=L.SMOOTH_MUL, rotate=mode == 1,
                         encode=L.ENC_NONE, out_x=True)["x"].bfloat16()


def check_layer(x, w, s, mode, meta, codes):
    """x brought to the weight's space times the weight is x w^T, up to what the weight's own encode lost."""
    xt = to_weight_space(x, s, mode)
    y = serve.linear(xt, meta, codes)
    check_linear(xt, meta, codes, y)
    xs, ws = x.float() * s, w / s
    if mode == 1:
        xs, ws = codec.rotate64(xs.contiguous()), codec.rotate64(ws.contiguous())
    wq = values64(meta, codes)
    want = x.double() @ w.double().t()
    # the encode's loss; x's rounding to bf16; the fp32 scalings and rotations (sums of 64) of both sides; the result's
    lost = (xs.double() @ (wq - ws.double()).t()).abs()
    tol = lost + (2 * BF16 + 200 * 2.0 ** -23) * (xs.double().abs() @ wq.abs().t()) + 200 * 2.0 ** -23 * (
        xs.double().abs() @ ws.double().abs().t()) + BF16 * want.abs()
    off = (y.double() - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.2f} of the tolerance"
    # and that is little: roundings have a variance of 1/12 of a step's square, a quad's peak is 3.5 steps or more, so
    # its mean square 3.5^2 / 4: under 3 percent (quads far below their group's peak lose more of less)
    assert (y.double() - want).square().mean() < 0.05 * want.square().mean()


@pytest.mark.parametrize("mode", [0, 1])
def test_product_in_a_smoothed_and_rotated_space(mode):
    T, N, C = 33, 200, 512
    x = torch.randn(T, C, generator=gen(70), device="cuda").bfloat16()
    x[:, ::50] *= 16
    w = torch.randn(N, C, generator=gen(71), device="cuda")
    s = x.float().abs().amax(0).clamp_min(0.1).rsqrt()
    p = codec.convert(w, kind=L.SRC_VALUES, smooth=s, smooth_mode=L.SMOOTH_DIV, rotate=mode == 1, dict5=False, packed=True)
    check_layer(x, w, s, mode, p["meta"], p["codes"])


@pytest.mark.parametrize("name", ["lin_c1024", "lin_c2560"])
def test_product_with_a_calibrated_weight(name, tmp_path):
    """calibrate_weight's result, and the same from the file that a conversion leaves."""
    import sys

    from conftest import GOLDEN
    if GOLDEN not in sys.path:
        sys.path.insert(0, GOLDEN)
    import pipeline_cases as pc

    from hif4x import linear, shard, weightset
    wpair, calib, tests, _ = pc.linear_inputs(name)
    dev = torch.device("cuda", torch.cuda.current_device())
    cuda = lambda pair: [t.cuda() for t in pair]  # noqa: E731
    path = weightset.convert_to_dir([(name, cuda(wpair), [cuda(c) for c in calib], cuda(tests[0]))], str(tmp_path))[name]
    rec = torch.load(path, weights_only=False)
    res = linear.calibrate_weight(wpair[0], wpair[1], calib)
    x, w = linear.decode_pair(tests[0], dev).bfloat16(), linear.decode_pair(wpair, dev)
    for packed_, st in ((rec["packed"].cuda(), rec["activation_state"]),
                        (shard.pack_params(res["weight_params"]), res["activation_state"])):
        meta, codes = shard.unpack_params(packed_, rec["rows"], rec["cols"])
        check_layer(x, w, st["s"].float().to(dev), st["mode"], meta, codes)
        # activations converted too: their values are bf16 numbers of the same space
        p = linear.dynamic_activation(*tests[0], st, return_device=True)
        xq = codec.decode(p, torch.bfloat16)
        check_linear(xq, meta, codes, serve.linear(xq, meta, codes))


def test_a_description_that_falls_reads_nothing_else():
    """cu_new must not fall; where it does all the same, the rows concerned are undefined, no place outside the call's
    tensors is touched, and the next call is right."""
    b = Batch([12, 12, 40], [9000, 9000, 9000], 1, 64, 16, 58)
    q = torch.randn(b.rows, 1, 64, generator=gen(59), device="cuda").bfloat16()
    bad = torch.tensor([0, 12, 4, 64], dtype=torch.int32, device="cuda")
    serve.paged_attention(q, b.cache, bad, b.len, b.pages)
    torch.cuda.synchronize()
    linalg.check_device_status()
    check_attention(b, q, serve.paged_attention(q, b.cache, *b.args))
    linalg.check_device_status()


def test_a_cache_takes_other_attributes():
    c = serve.PagedKV.empty(2, 16, 1, 64, "cuda")
    c.layer = 3
    assert c.layer == 3


def test_a_graph_of_both_kinds_with_other_lengths():
    """One captured call, replayed with descriptions that make every sequence single tokens, chunks or nothing in
    turn: each replay is right, and equal to an eager call of the same sizes."""
    kvh, dh, page, rows, qh = 2, 128, 32, 90, 8
    cases = [([1, 80, 2, 7], [9000, 4000, 5000, 9000]), ([80, 1, 9, 0], [9000, 30, 9000, 7000]),
             ([0, 0, 90, 0], [1, 1, 6000, 1]), ([4, 4, 4, 4], [9000, 8000, 7000, 3]), ([1, 1, 1, 1], [9000, 2, 5000, 4097])]
    b = Batch([20] * 4, [9000] * 4, kvh, dh, page, 57)
    q = torch.randn(rows, qh, dh, generator=gen(58), device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve.paged_attention(q, b.cache, *b.args)
    torch.cuda.current_stream().wait_stream(side)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serve.paged_attention(q, b.cache, *b.args, out=out)
    for new, lens in cases + cases[::-1]:
        b.new, b.lens, b.rows = new, lens, sum(new)
        b.cu.copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
        b.len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        assert (out[b.rows:] == 5).all()
        check_attention(b, q, out)
        assert torch.equal(out[:b.rows], serve.paged_attention(q, b.cache, *b.args)[:b.rows])
    linalg.check_device_status()


