"""Sliding-window attention on the CPU: the rule itself, packed documents, rows that see nothing, gradients, refusals."""
import math

import pytest
import torch

from maltos_b200.ops.attention import attention, build_window_mask, sliding_window_attention


def _rule(Sq, Sk, window, sinks, ids=None):
    """The rule written out pair by pair."""
    seen = torch.zeros(Sq, Sk, dtype=torch.bool)
    for i in range(Sq):
        p = i + Sk - Sq
        if p < 0 or (ids is not None and ids[p] == -1):
            continue
        s = p
        while ids is not None and s > 0 and ids[s - 1] == ids[p]:
            s -= 1
        if ids is None:
            s = 0
        for j in range(s, p + 1):
            seen[i, j] = p - j < window or j - s < sinks
    return seen


@pytest.mark.parametrize("Sq,Sk,window,sinks", [(1, 1, 1, 0), (9, 9, 3, 0), (9, 9, 3, 2), (4, 11, 5, 1), (1, 8, 2, 3), (6, 4, 2, 1), (7, 7, 100, 100)])
def test_mask_is_the_rule(Sq, Sk, window, sinks):
    assert torch.equal(build_window_mask(Sq, Sk, window, sinks)[0], _rule(Sq, Sk, window, sinks))


@pytest.mark.parametrize("ids", [[0, 0, 0, 1, 1, 2, 2, 2, 2], [-1, 3, 3, 3, -1, -1, 5, 5, -1], [7] * 9, [-1] * 9, [0, 0, 1, 1, 0, 0, 0, -1, 0]])
@pytest.mark.parametrize("Sq,window,sinks", [(9, 2, 0), (9, 2, 1), (4, 3, 2), (12, 2, 1)])
def test_mask_with_documents_is_the_rule(ids, Sq, window, sinks):
    t = torch.tensor([ids])
    assert torch.equal(build_window_mask(Sq, 9, window, sinks, t)[0], _rule(Sq, 9, window, sinks, ids))


def test_window_of_the_whole_row_is_causal_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 13, h, 8, generator=g) for h in (4, 2, 2))
    out, lse = sliding_window_attention(q, k, v, window=13, return_lse=True)
    ref, ref_lse = attention(q, k, v, causal=True, return_lse=True)
    # the same sums in fp32 in another order: 13 terms of eps/2 each
    torch.testing.assert_close(out, ref, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(lse, ref_lse, rtol=1e-5, atol=1e-5)


def test_rows_that_see_nothing_are_zero_and_give_no_gradient():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 6, 2, 8, generator=g, dtype=torch.float64).requires_grad_() for _ in range(3))
    ids = torch.tensor([[-1, 0, 0, -1, 1, -1]])
    out, lse = sliding_window_attention(q, k, v, window=2, sinks=1, sequence_ids=ids, return_lse=True)
    pad = ids[0] == -1
    assert out[0, pad].abs().max() == 0 and torch.isneginf(lse[0, :, pad]).all()
    out.sum().backward()
    for t in (q, k, v):
        assert torch.isfinite(t.grad).all() and t.grad[0, pad].abs().max() == 0
    more = sliding_window_attention(torch.randn(1, 5, 2, 8), torch.randn(1, 2, 2, 8), torch.randn(1, 2, 2, 8), window=2)
    assert more[:, :3].abs().max() == 0 and more[:, 3:].abs().min() > 0


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 7, h, 4, generator=g, dtype=torch.float64).requires_grad_() for h in (4, 2, 2))
    ids = torch.tensor([[0, 0, 0, 0, 1, 1, -1]])
    assert torch.autograd.gradcheck(lambda a, b, c: sliding_window_attention(a, b, c, window=2, sinks=1, sequence_ids=ids), (q, k, v))


@pytest.mark.parametrize("B,Sq,Sk", [(0, 3, 3), (1, 0, 3), (1, 3, 0)])
def test_lengths_of_zero(B, Sq, Sk):
    q, k = torch.randn(B, Sq, 2, 8, requires_grad=True), torch.randn(B, Sk, 1, 8)
    out, lse = sliding_window_attention(q, k, k, window=2, return_lse=True)
    assert out.shape == q.shape and lse.shape == (B, 2, Sq)
    assert out.numel() == 0 or (out.abs().max() == 0 and torch.isneginf(lse).all())


def test_refusals():
    q, k = torch.randn(2, 6, 4, 8), torch.randn(2, 6, 2, 8)
    ids = torch.zeros(2, 6, dtype=torch.int64)
    bad = [
        (dict(window=0), "window"), (dict(window=2.0), "window"), (dict(window=True), "window"), (dict(window=2, sinks=-1), "sinks"),
        (dict(window=2, scale=0.0), "scale"), (dict(window=2, scale=math.inf), "scale"), (dict(window=2, sequence_ids=ids[:, :5]), "sequence_ids"),
        (dict(window=2, sequence_ids=ids.float()), "sequence_ids"),
    ]
    for kw, what in bad:
        with pytest.raises(ValueError, match=what):
            sliding_window_attention(q, k, k, **kw)
    with pytest.raises(ValueError, match="multiple"):
        sliding_window_attention(q[:, :, :3], k, k, window=2)
    with pytest.raises(ValueError, match="type"):
        sliding_window_attention(q, k.half(), k.half(), window=2)
    with pytest.raises(ValueError, match="takes q"):
        sliding_window_attention(q, k, k[:, :5], window=2)
