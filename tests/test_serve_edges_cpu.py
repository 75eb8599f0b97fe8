"""Host side of the serving operators at the edges (no GPU calls): which tensors lie over one another."""
import itertools

import pytest
import torch

pytest.importorskip("hif4x._lib")
from hif4x import serve  # noqa: E402


def views():
    """(view, its element numbers) of one buffer of 240 elements: column ranges, rows, heads, one element."""
    base, at = torch.zeros(240, dtype=torch.bfloat16), torch.arange(240)
    cuts = [lambda t: t.view(10, 24)[:, :8], lambda t: t.view(10, 24)[:, 8:20], lambda t: t.view(10, 24)[:, 16:],
            lambda t: t.view(10, 24)[2:5, 4:12], lambda t: t.view(10, 24)[:1, 8:16], lambda t: t.view(10, 24)[5:],
            lambda t: t.view(20, 12)[:, :4], lambda t: t.view(10, 3, 8)[:, 1], lambda t: t.view(5, 2, 4, 6)[:, 0],
            lambda t: t.view(5, 2, 4, 6)[:, 1, 1:3], lambda t: t.view(5, 2, 4, 6)[1:, 1, :, 2:4],
            lambda t: t.view(3, 80)[:, 8:24].unflatten(1, (2, 8)).transpose(0, 1), lambda t: t[7:8], lambda t: t[100:140],
            lambda t: t.view(10, 24)[::2, :8], lambda t: t.view(10, 24)[1::2, :8], lambda t: t.view(10, 24).t()[:4]]
    return [(c(base), set(c(at).reshape(-1).tolist())) for c in cuts]


def test_apart_is_right_about_views_of_one_buffer():
    """No pair that shares an element passes, and column ranges of one pitch that share none do."""
    passed = 0
    for (a, ea), (b, eb) in itertools.product(views(), repeat=2):
        free = not serve._overlap(a, b) or serve._beside(a, b)
        assert not (free and ea & eb)
        passed += free and serve._overlap(a, b)
        if not ea & eb and serve._runs(a)[0] == serve._runs(b)[0] > 0:
            assert free, (a.shape, a.stride(), b.shape, b.stride())
    assert passed > 10
