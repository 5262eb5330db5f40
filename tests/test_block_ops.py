"""Scaled embedding and block norm on the CPU: formulas, gradients against differences, sizes of zero, refusals."""
import pytest
import torch
import torch.nn.functional as F

from maltos_b200.ops import _lib
from maltos_b200.ops.embedding import ScaledEmbedding, embedding
from maltos_b200.ops.norm import add_rms_norm, block_norm


def _tensors(shape, H, *, gate, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()   # noqa: E731
    return mk(*shape), mk(*shape), mk(H), mk(H), None if gate is None else mk(*(shape if gate == "element" else (H,)))


@pytest.mark.parametrize("gate", [None, "channel", "element"])
@pytest.mark.parametrize("after,before", [(True, True), (True, False), (False, True), (False, False)])
def test_block_norm_gradients_against_differences(gate, after, before):
    x, r, w1, w2, g = _tensors((2, 3, 6), 6, gate=gate)
    used = [t for t in (x, r, w1 if after else None, w2 if before else None, g) if t is not None]

    def f(*_):
        return block_norm(x, r, w1 if after else None, w2 if before else None, gate=g, scale=0.3, eps=1e-3)

    assert torch.autograd.gradcheck(f, used)


def test_block_norm_is_the_formula():
    x, r, w1, w2, g = _tensors((4, 6), 6, gate="channel")
    y, h = block_norm(x, r, w1, w2, gate=g, scale=0.25, eps=1e-6)
    want = r + 0.25 * g * w1 * x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    torch.testing.assert_close(h, want)
    torch.testing.assert_close(y, w2 * want / (want.square().mean(-1, keepdim=True) + 1e-6).sqrt())
    a, b = block_norm(x.float(), r.float(), None, w2.float()), add_rms_norm(x.float(), r.float(), w2.float())
    torch.testing.assert_close(a[0], b[0])
    torch.testing.assert_close(a[1], b[1])


def test_block_norm_without_elements():
    e = torch.zeros(0, 8, requires_grad=True)
    y, h = block_norm(e, e, torch.ones(8), torch.ones(8))
    assert y.shape == h.shape == (0, 8)


def test_block_norm_refusals():
    x, w = torch.randn(2, 8), torch.ones(8)
    for args, kw, what in [((x, x[:1], w), {}, "one shape"), ((x, x.double(), w), {}, "residual"), ((x, x, w[:4]), {}, "weight"),
                           ((x, x, w, w[:4]), {}, "next_weight"), ((x, x, w), dict(gate=torch.ones(2, 1)), "gate"),
                           ((x, x, w.double()), {}, "weight"), ((x, x, w), dict(scale=float("nan")), "finite"), ((x, x, w), dict(eps=-1.0), "eps"),
                           ((x.long(), x.long(), None), {}, "floating")]:
        with pytest.raises(ValueError, match=what):
            block_norm(*args, **kw)


@pytest.mark.parametrize("scale,pad", [(1.0, None), (2.5, None), (0.5, 3)])
def test_embedding_matches_torch(scale, pad):
    w = torch.randn(11, 6, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[3, 0, 10], [3, 3, 7]])
    out = embedding(ids, w, scale=scale, padding_idx=pad)
    d = torch.randn_like(out)
    ref = F.embedding(ids, w, padding_idx=pad) * scale
    assert torch.equal(out, ref)
    assert torch.equal(torch.autograd.grad(out, w, d)[0], torch.autograd.grad(ref, w, d)[0])


def test_scaled_embedding_module():
    torch.manual_seed(0)
    m = ScaledEmbedding(9, 4, 3.0)
    assert list(m.state_dict()) == ["weight"] and isinstance(m, torch.nn.Embedding)
    ids = torch.tensor([1, 8])
    assert torch.equal(m(ids), F.embedding(ids, m.weight) * 3.0)
    assert m(ids[:0]).shape == (0, 4)


def test_embedding_refusals():
    w, ids = torch.randn(5, 4), torch.tensor([0, 1])
    for args, kw, what in [((ids.float(), w), {}, "int32 or int64"), ((ids, w[0]), {}, "matrix"), ((ids, w.long()), {}, "matrix"),
                           ((ids, w), dict(scale=float("inf")), "finite"), ((ids, w), dict(padding_idx=5), "padding_idx"),
                           ((ids, w), dict(padding_idx=-1), "padding_idx")]:
        with pytest.raises(ValueError, match=what):
            embedding(*args, **kw)
    with pytest.raises(IndexError):
        embedding(torch.tensor([5]), w)


def test_entry_points_refuse_sizes_before_touching_the_device():
    """Sizes whose launches would not fit the grid (2^21 columns and more are 65536 blocks of the narrowest join) and sizes that no
    kernel takes come back as errors; no pointer is read."""
    lib = _lib.lib()
    a = 4096
    for tokens, H, rows in ((1, 2 ** 21 + 1, 4), (0, 8, 4), (2 ** 31, 8, 4), (1, 0, 4), (1, 8, 0), (1, 8, 2 ** 31)):
        assert lib.mb_embedding_fwd(a, 1, a, a, 0, tokens, H, rows, 1.0, None) == -1
        assert lib.mb_embedding_bwd(a, 1, a, a, a, 0, tokens, H, rows, -1, 1.0, None) == -1
    assert lib.mb_embedding_bwd(a, 1, a, a, a, 3, 1, 8, 4, -1, 1.0, None) == -1          # no such type
    for rows, H in ((0, 8), (1, 4), (1, 12), (1, 16392), (2 ** 31, 8)):
        assert lib.mb_block_norm_fwd(a, a, None, None, None, 0, a, None, None, None, 0, rows, H, 1.0, 1e-6, None) == -1
        assert lib.mb_block_norm_bwd(None, a, None, None, None, None, None, 0, None, None, a, a, None, None, None, None, None, 0, rows, H, 1.0, None) == -1
    assert lib.mb_block_norm_fwd(a + 8, a, None, None, None, 0, a, None, None, None, 0, 1, 8, 1.0, 1e-6, None) == -1     # 8 bytes off
