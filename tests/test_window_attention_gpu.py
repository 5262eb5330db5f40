"""The sliding-window kernels against the rule in 64 bits, element by element. The bounds count roundings (u = 2^-8, half a bf16
step) and are derived beside them; nothing else of size takes part: scores, sums and exponentials are fp32, whose own errors
are covered by the factor 1.05 and 2^-12 of the sum of magnitudes."""
import math

import pytest
import torch

from maltos_b200.ops import _lib
from maltos_b200.ops.attention import build_window_mask, sliding_window_attention
from maltos_b200.ops.window_attn import document_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


def _qkv(B, Sq, Sk, Hq, Hkv, D, seed=0, packed=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if packed:
        t = torch.randn(B, Sk, Hq + 2 * Hkv, D, device=DEV, generator=g).bfloat16()
        return t[:, Sk - Sq:, :Hq], t[:, :, Hq:Hq + Hkv], t[:, :, Hq + Hkv:]
    mk = lambda s, h: torch.randn(B, s, h, D, device=DEV, generator=g).bfloat16()   # noqa: E731
    return mk(Sq, Hq), mk(Sk, Hkv), mk(Sk, Hkv)


def _documents(B, S, lengths, pad_first=0):
    ids = torch.full((B, S), -1, dtype=torch.int64, device=DEV)
    for b in range(B):
        at = pad_first + 3 * b
        for n, length in enumerate(lengths):
            ids[b, at:at + length] = n
            at += length + (1 if n % 2 else 0)     # now and then a padding token between documents
    return ids


def _expect(q, k, v, dout, window, sinks, ids, scale):
    """Values and bounds of (out, lse, dq, dk, dv), from the formulas in 64 bits."""
    B, Sq, hq, D = q.shape
    Sk, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    heads = lambda t: t.double().permute(0, 2, 1, 3)                         # noqa: E731
    Q, dO = heads(q), heads(dout)
    K, V = heads(k).repeat_interleave(g, 1), heads(v).repeat_interleave(g, 1)
    seen = build_window_mask(Sq, Sk, window, sinks, ids, q.device)[:, None]
    S = (Q @ K.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(S, -1)
    P = torch.exp(S - lse.masked_fill(lse == -math.inf, 0.0).unsqueeze(-1))
    out = P @ V
    # The weights are rounded to bf16 (u of each) and divided by the sum of the rounded ones (u again at most); the result is
    # rounded once more, for the backward it is kept to 2^-16.
    e_p = 1.05 * 2 * U + 2.0 ** -12
    e_out = e_p * (P @ V.abs())
    b_out = e_out + U * (out.abs() + e_out)
    dP = dO @ V.transpose(-1, -2)
    delta = (dO * out).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    # delta is taken from that output; dS is formed from rounded weights and rounded to bf16
    e_delta = (dO.abs() * e_out).sum(-1, keepdim=True) + 2.0 ** -12 * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    e_ds = P * e_delta + (e_p + 1.05 * U) * dS.abs() + 2.0 ** -12 * P * (dO.abs() @ V.abs().transpose(-1, -2))
    fold = lambda t: t.reshape(B, hkv, g, Sk, D).sum(2)                      # noqa: E731
    dq, e_dq = scale * dS @ K, scale * e_ds @ K.abs()
    dk, e_dk = fold(scale * dS.transpose(-1, -2) @ Q), fold(scale * e_ds.transpose(-1, -2) @ Q.abs())
    dv, e_dv = fold(P.transpose(-1, -2) @ dO), fold(e_p * P.transpose(-1, -2) @ dO.abs())
    pack = lambda val, err: (val.permute(0, 2, 1, 3), (err + U * (val.abs() + err)).permute(0, 2, 1, 3))   # noqa: E731
    return (out.permute(0, 2, 1, 3), b_out.permute(0, 2, 1, 3)), lse, pack(dq, e_dq), pack(dk, e_dk), pack(dv, e_dv)


def _near(name, got, want):
    value, bound = want
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    over = (got.double() - value).abs() - bound - 1e-9
    assert over.max().item() <= 0, f"{name}: {over.max().item():.3g} over its bound at {tuple(int(i) for i in torch.nonzero(over == over.max())[0])}"


def _case(B, Sq, Sk, Hq, Hkv, D, window, sinks, ids=None, seed=0, packed=False, scale=None):
    q, k, v = (t.detach().requires_grad_() for t in _qkv(B, Sq, Sk, Hq, Hkv, D, seed, packed))
    dout = torch.randn(B, Sq, Hq, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed + 1)).bfloat16()
    out, lse = sliding_window_attention(q, k, v, window=window, sinks=sinks, sequence_ids=ids, return_lse=True, scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    _lib.fetch_status()
    w_out, w_lse, *w_grads = _expect(q.detach(), k.detach(), v.detach(), dout, window, sinks, ids, scale or 1 / math.sqrt(D))
    _near("out", out.detach(), w_out)
    finite = torch.isfinite(w_lse)
    assert torch.equal(torch.isfinite(lse), finite) and torch.isneginf(lse[~finite]).all()
    # scores are sums of D fp32 products of magnitude up to ~6 sigma: 2^-24 * D * |s| stays below 1e-4
    assert not finite.any() or (lse[finite].double() - w_lse[finite]).abs().max() < 1e-4
    for name, got, want in zip(("dq", "dk", "dv"), grads, w_grads):
        _near(name, got, want)
    return out.detach(), lse, grads


@pytest.mark.parametrize("S,window,sinks", [(1, 1, 0), (2, 1, 1), (127, 64, 0), (128, 128, 4), (129, 1, 0), (200, 129, 1), (300, 100, 4), (513, 64, 130),
                                            (513, 128, 200), (640, 1000, 7), (1000, 257, 0), (1000, 256, 16)])
@pytest.mark.parametrize("D", [64, 128])
def test_square(S, window, sinks, D):
    _case(1, S, S, 2, 2, D, window, sinks)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (4, 1), (6, 2), (8, 2), (5, 5)])
def test_groups(Hq, Hkv):
    _case(2, 333, 333, Hq, Hkv, 64, 90, 5)


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 128), (15, 5, 64), (15, 15, 128)])
def test_two_tiles_to_an_item(Hq, Hkv, D):
    """More tiles than SMs: items of two heads (even groups) or of two neighbouring row tiles, several items to a CTA."""
    _case(3, 700, 700, Hq, Hkv, D, 150, 3)


@pytest.mark.parametrize("Sq,Sk,window,sinks", [(1, 1, 1, 0), (1, 700, 256, 4), (1, 700, 900, 0), (1, 129, 1, 1), (77, 500, 130, 9), (128, 131, 64, 0),
                                                (300, 900, 128, 200), (300, 140, 64, 2), (257, 1, 4, 1)])
def test_other_lengths(Sq, Sk, window, sinks):
    _case(2, Sq, Sk, 4, 2, 128, window, sinks)


@pytest.mark.parametrize("lengths,pad", [([40, 200, 1, 300, 60], 0), ([640], 0), ([128, 128, 128, 128, 100], 5), ([3] * 50, 130), ([500], 64), ([], 0)])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 4), (1, 1), (200, 140), (1000, 0)])
def test_documents(lengths, pad, window, sinks):
    _case(2, 643, 643, 4, 2, 64, window, sinks, ids=_documents(2, 643, lengths, pad))


@pytest.mark.parametrize("Hq,Hkv", [(14, 7), (16, 16), (8, 1)])
def test_documents_with_two_tiles_to_an_item(Hq, Hkv):
    _case(3, 1290, 1290, Hq, Hkv, 64, 100, 6, ids=_documents(3, 1290, [400, 129, 5, 600], 7).to(torch.int32))


def test_documents_of_a_chunk():
    _case(2, 150, 643, 4, 2, 64, 60, 3, ids=_documents(2, 643, [300, 330]))


def test_an_id_that_returns_begins_another_document():
    ids = torch.tensor([[0] * 100 + [1] * 100 + [0] * 100], device=DEV)
    _case(1, 300, 300, 2, 1, 64, 260, 2, ids=ids)


def test_document_bounds():
    for S in (1, 5, 1024, 1025, 5000):
        ids = torch.randint(-1, 2, (3, S), device=DEV, generator=torch.Generator(device=DEV).manual_seed(S))
        ids[2] = 4
        for t in (ids, ids.to(torch.int32)):
            starts, ends = document_bounds(t)
            for b in range(3):
                row, s = ids[b].tolist(), 0
                want_s, want_e = [], [0] * S
                for j in range(S):
                    if j and row[j] != row[j - 1]:
                        s = j
                    want_s.append(2 ** 31 - 1 if row[j] == -1 else s)
                e = S
                for j in reversed(range(S)):
                    want_e[j] = 0 if row[j] == -1 else e
                    if j and row[j] != row[j - 1]:
                        e = j
                assert starts[b].tolist() == want_s and ends[b].tolist() == want_e


def test_strided_inputs_and_scale():
    _case(2, 260, 260, 6, 3, 128, 70, 2, packed=True, scale=0.05)
    q, k, v = _qkv(2, 200, 200, 4, 2, 64)
    plain = sliding_window_attention(q, k, v, window=33, sinks=2)
    bhsd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]           # heads outside tokens: copied
    assert torch.equal(plain, sliding_window_attention(*bhsd, window=33, sinks=2))
    wide = [torch.cat([t, t[..., :4]], -1)[..., :64] for t in (q, k, v)]                 # rows of 68 elements: copied
    assert torch.equal(plain, sliding_window_attention(*wide, window=33, sinks=2))
    one = [t[:1].expand(2, -1, -1, -1) for t in (q, k, v)]                               # broadcast batch
    assert torch.equal(sliding_window_attention(*one, window=33)[0], sliding_window_attention(*one, window=33)[1])
    leaf = [t.detach().requires_grad_() for t in (q, k, v)]
    sliding_window_attention(*leaf, window=33).float().sum().backward()                  # a broadcast output gradient
    assert all(torch.isfinite(t.grad).all() for t in leaf)


def test_same_bits_every_time():
    ids = _documents(2, 643, [300, 330])
    a = _case(2, 643, 643, 8, 1, 64, 100, 4, ids=ids)
    b = _case(2, 643, 643, 8, 1, 64, 100, 4, ids=ids)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


def test_large_scores_and_rising_maxima():
    """Row maxima that rise by far more than 2^8 from block to block, and scores of a few hundred."""
    B, S, H, D = 1, 600, 2, 64
    q, k, v = _qkv(B, S, S, H, H, D)
    k = (k.float() * torch.linspace(0.1, 20, S, device=DEV).view(1, S, 1, 1)).bfloat16()
    out = sliding_window_attention(q, k, v, window=300, sinks=4)
    (value, bound), _, *_ = _expect(q, k, v, torch.zeros_like(q), 300, 4, None, 1 / 8)
    # scores up to ~200 in fp32: 64 products, relative 2^-18 of the sum of magnitudes, so exp is off by up to 2e-3
    _near("out", out, (value, bound + 4e-3 * v.float().abs().max()))


def test_streams_and_captured_graphs():
    q, k, v = (t.requires_grad_() for t in _qkv(2, 300, 300, 4, 2, 64))
    dout = torch.randn_like(q)
    ids = _documents(2, 300, [100, 150])

    def step():
        out = sliding_window_attention(q, k, v, window=70, sinks=2, sequence_ids=ids)
        return (out, *torch.autograd.grad(out, (q, k, v), dout))

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for t in held:
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))
    _lib.fetch_status()


def test_activation_checkpointing_replays_the_forward():
    from torch.utils.checkpoint import checkpoint

    from maltos_b200.utils.activation_checkpoint import activation_checkpoint_context_fn

    q, k, v = (t.requires_grad_() for t in _qkv(1, 300, 300, 4, 2, 64))
    f = lambda a: sliding_window_attention(a * 1.0, k, v, window=70, sinks=2)           # noqa: E731
    plain = torch.autograd.grad(f(q).float().square().sum(), (q, k, v))
    kept = torch.autograd.grad(checkpoint(f, q, use_reentrant=False, context_fn=activation_checkpoint_context_fn).float().square().sum(), (q, k, v))
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))


def test_other_types_and_head_sizes_run_the_restatement():
    for dtype, D in ((torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 32), (torch.bfloat16, 96)):
        q, k, v = (t[..., :D].to(dtype).contiguous() for t in _qkv(1, 70, 70, 2, 1, 128))
        out = sliding_window_attention(q, k, v, window=20, sinks=2)
        (value, _), *_ = _expect(q, k, v, torch.zeros_like(q), 20, 2, None, 1 / math.sqrt(D))
        eps = torch.finfo(dtype).eps
        assert out.dtype == dtype and (out.double() - value).abs().max() <= (eps / 2 + 2e-6) * 4 + 1e-5


@pytest.mark.parametrize("Sq,Sk,Hq,Hkv,D,window,sinks", [(1, 1, 1, 1, 64, 1, 0), (1, 700, 8, 2, 128, 300, 4), (1, 700, 4, 4, 64, 1000, 0), (2, 517, 6, 2, 128, 100, 130),
                                                         (1, 5000, 16, 2, 64, 4096, 16), (3, 33, 10, 1, 128, 7, 2), (8, 400, 4, 1, 64, 60, 3),
                                                         (5, 3, 2, 1, 128, 2, 1), (1, 1300, 32, 1, 128, 1200, 4), (4, 200, 12, 4, 128, 1, 0)])
def test_few_queries_without_gradients(Sq, Sk, Hq, Hkv, D, window, sinks):
    ids = _documents(3, Sk, [Sk // 2, Sk // 3], 1) if Sk > 30 else None
    for seq in (None, ids):
        for packed in (False, True):
            if packed and Sq > Sk:
                continue
            q, k, v = _qkv(3, Sq, Sk, Hq, Hkv, D, seed=Sk, packed=packed)
            with torch.no_grad():
                out, lse = sliding_window_attention(q, k, v, window=window, sinks=sinks, sequence_ids=seq, return_lse=True)
            _lib.fetch_status()
            (value, bound), w_lse, *_ = _expect(q, k, v, torch.zeros_like(q), window, sinks, seq, 1 / math.sqrt(D))
            _near("out", out, (value, bound))
            finite = torch.isfinite(w_lse)
            assert torch.equal(torch.isfinite(lse), finite) and torch.isneginf(lse[~finite]).all()
            assert not finite.any() or (lse[finite].double() - w_lse[finite]).abs().max() < 1e-4
            again = sliding_window_attention(q, k, v, window=window, sinks=sinks, sequence_ids=seq)
            assert torch.equal(out, again)
