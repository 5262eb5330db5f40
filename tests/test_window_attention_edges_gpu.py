"""Sliding-window attention where its ordinary cases do not reach. Oracle and bounds: test_window_attention_gpu."""
import math

import pytest
import torch

from maltos_b200.ops import _lib
from maltos_b200.ops.attention import build_window_mask, sliding_window_attention, sliding_window_reference
from tests.test_window_attention_gpu import DEV, U, _case, _documents, _expect, _qkv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("Sq,Hq,Hkv,D", [(1, 8, 1, 128), (2, 4, 2, 64), (300, 4, 2, 128), (300, 3, 3, 64)])
def test_a_query_that_is_no_number_spoils_its_own_row_only(Sq, Hq, Hkv, D, keep):
    """NaN and infinity in a query give NaN, in tiles, for few queries and in a training forward; "sees nothing" stays zero and -inf."""
    Sk = 300
    q, k, v = _qkv(3, Sq, Sk, Hq, Hkv, D, seed=Sq)
    ids = torch.zeros(3, Sk, dtype=torch.int64, device=DEV)
    ids[2] = -1
    clean = q.clone()
    q[0, Sq - 1, 1, 5] = float("nan")
    q[1, Sq - 1, 0, 2] = float("inf")
    q[1, Sq - 1, 2, 7] = float("-inf")
    q[2, 0, 1, 0] = float("nan")                   # of a row of padding: zero all the same
    bad = torch.zeros(3, Sq, Hq, dtype=torch.bool, device=DEV)
    bad[0, Sq - 1, 1] = bad[1, Sq - 1, 0] = bad[1, Sq - 1, 2] = True
    leaf = q.requires_grad_() if keep else q
    out, lse = sliding_window_attention(leaf, k, v, window=120, sinks=4, sequence_ids=ids, return_lse=True)
    _lib.fetch_status()
    out, lse = out.detach(), lse.transpose(1, 2)
    assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad)
    assert torch.isnan(lse[0, Sq - 1, 1]) and not torch.isfinite(lse[bad]).any() and not torch.isneginf(lse[bad]).any()
    assert out[2].abs().max() == 0 and torch.isneginf(lse[2]).all()
    want = sliding_window_reference(q.detach(), k, v, window=120, sinks=4, sequence_ids=ids)
    assert torch.equal(torch.isnan(want).any(-1), bad)
    (value, bound), w_lse, *_ = _expect(clean, k, v, torch.zeros_like(clean), 120, 4, ids, 1 / math.sqrt(D))
    assert ((out.double() - value).abs() - bound)[~bad].max() <= 1e-9
    good = ~bad[:2]
    assert (lse[:2][good].double() - w_lse.transpose(1, 2)[:2][good]).abs().max() < 1e-4


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[2900], [1000, 30, 1700, 5, 200], [1400, 1400]])
def test_long_documents_whose_first_blocks_are_cut(lengths, D):
    """Long lists of queries of the blocks that hold first tokens, of one head (pieces for want of blocks) and of many."""
    ids = _documents(1, 3001, lengths, 40)
    _case(1, 3001, 3001, 2, 1, D, 64, 4, ids=ids)
    _case(1, 3001, 3001, 10, 10, D, 130, 200, ids=ids)


@pytest.mark.parametrize("packed", [False, True])
def test_more_key_blocks_than_the_list_takes_at_a_time(packed):
    """1120 key blocks, the first of each row cut into pieces; rows on both sides of the list's steps against the formula."""
    B, S, D, window, sinks = 70, 2000, 64, 64, 4
    q, k, v = (t.requires_grad_() for t in _qkv(B, S, S, 1, 1, D, seed=3))
    ids = _documents(B, S, [700, 1000], 0) if packed else None
    dout = torch.randn(B, S, 1, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)).bfloat16()
    out = sliding_window_attention(q, k, v, window=window, sinks=sinks, sequence_ids=ids)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    _lib.fetch_status()
    for b in (0, 62, 63, 64, 69):
        at = slice(b, b + 1)
        w_out, _, *w_grads = _expect(*(t.detach()[at] for t in (q, k, v)), dout[at], window, sinks, None if ids is None else ids[at], 1 / math.sqrt(D))
        for got, (value, bound) in zip((out.detach(), *grads), (w_out, *w_grads)):
            assert ((got[at].double() - value).abs() - bound).max() <= 1e-9


@pytest.mark.parametrize("D", [64, 128])
def test_without_first_tokens_no_block_before_the_window_is_read(D):
    """A document that starts inside a block, and a value in that block that only the rows near it may see: NaN tells who reads it."""
    q, k, v = _qkv(1, 643, 643, 4, 2, D)
    ids = _documents(1, 643, [560], 70)
    dout = torch.randn_like(q)

    def run(v):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = sliding_window_attention(*leaves, window=50, sequence_ids=ids)
        return out.detach(), torch.autograd.grad(out, leaves, dout)[0]

    want = run(v)
    v[0, 72] = float("nan")
    for got, clean in zip(run(v), want):
        assert torch.isnan(got[0, 72:122]).all()
        assert torch.equal(got[0, 256:], clean[0, 256:])      # the row tiles whose windows begin in a later block


@pytest.mark.parametrize("D,lean_k,lean_q", [(64, 12.0, 8.0), (128, 20.0, 6.0)])
def test_dq_of_rows_whose_weight_is_on_the_first_token(D, lean_k, lean_q):
    """Queries lean towards what the first key holds, as trained models' do: nearly all weight is on one key, and dS there is the small
    difference dP - delta, so an error e of delta comes out as e * scale * sum P k, far larger than dq's other errors.

    Bound of the norm of dq's error. Weights and dS are rounded to bf16, each off by at most u, relative and independent, so of
    variance u^2 / 3 at most. With delta taken from the same weights the former enter as
    sum_j dS_j d_j (k_j - sum P k), the latter as sum_j dS_j d_j k_j; twice the root of the summed variances, and dq's own rounding.
    What delta from the rounded output alone would add is far outside, which is asserted too."""
    S, W, N = 300, 100, 1
    scale = 1 / math.sqrt(D)
    g = torch.Generator(device=DEV).manual_seed(D)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)                # noqa: E731
    lean = torch.nn.functional.normalize(rnd(D), dim=0)
    q = (rnd(1, S, 2, D) + lean_q * lean).bfloat16().requires_grad_()
    k = rnd(1, S, 2, D)
    k[:, :1] += lean_k * lean
    k, v, dout = k.bfloat16().requires_grad_(), rnd(1, S, 2, D).bfloat16().requires_grad_(), rnd(1, S, 2, D).bfloat16()
    out = sliding_window_attention(q, k, v, window=W, sinks=N)
    dq = torch.autograd.grad(out, (q, k, v), dout)[0]
    _lib.fetch_status()
    Q, K, V, dO = (t.detach()[0].double().transpose(0, 1) for t in (q, k, v, dout))
    seen = build_window_mask(S, S, W, N, None, DEV)
    P = (Q @ K.transpose(1, 2) * scale).masked_fill(~seen, -math.inf).softmax(-1)
    O, dP = P @ V, dO @ V.transpose(1, 2)
    delta = (dO * O).sum(-1, keepdim=True)
    dS, mean_k = P * (dP - delta), P @ K
    exact = scale * dS @ K
    spread = ((K.unsqueeze(1) - mean_k.unsqueeze(2)).square() + K.unsqueeze(1).square()).sum(-1)
    bound = 2 * scale * U / math.sqrt(3) * (dS.square() * spread).sum().sqrt() + U / math.sqrt(3) * exact.norm()
    from_out = scale * ((dO * O.bfloat16().double()).sum(-1, keepdim=True) - delta) * mean_k
    assert from_out.norm() > 3 * bound
    assert (dq[0].double().transpose(0, 1) - exact).norm() <= bound


@pytest.mark.parametrize("lengths,pad", [([40, 200, 1, 300, 60], 0), ([128, 128, 128, 128, 100], 5), ([3] * 50, 130), ([], 0)])
@pytest.mark.parametrize("window,sinks,Hq,Hkv", [(50, 0, 4, 2), (50, 4, 3, 3), (200, 140, 4, 1)])
def test_documents_at_head_dim_128(lengths, pad, window, sinks, Hq, Hkv):
    _case(2, 643, 643, Hq, Hkv, 128, window, sinks, ids=_documents(2, 643, lengths, pad))


def test_documents_in_captured_graphs_that_share_a_pool():
    """Two graphs of the same memory pool, replayed in turn with other documents each time."""
    q, k, v = (t.requires_grad_() for t in _qkv(1, 700, 700, 4, 2, 64))
    dout = torch.randn_like(q)
    layouts = [_documents(1, 700, lengths) for lengths in ([300, 390], [40, 600], [650])]
    ids = [layouts[0].clone(), layouts[0].clone()]

    def step(i):
        out = sliding_window_attention(q, k, v, window=70, sinks=2, sequence_ids=i)
        return (out, *torch.autograd.grad(out, (q, k, v), dout))

    want = [[t.detach().clone() for t in step(i)] for i in layouts]
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = step(ids[0])
    with torch.cuda.graph(second, pool=first.pool()):
        b = step(ids[1])
    for i, j in ((0, 1), (2, 0), (1, 2)):
        ids[0].copy_(layouts[i])
        first.replay()
        got = [t.detach().clone() for t in a]
        ids[1].copy_(layouts[j])
        second.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want[i])) and all(torch.equal(x, y) for x, y in zip(b, want[j]))
    _lib.fetch_status()


@pytest.mark.parametrize("D", [64, 128])
def test_weights_of_the_backward_over_their_whole_range(D):
    """With unit vectors as the output's gradient, dV holds the backward's weights themselves, from near 1 to below the smallest normal
    number, in every column of a tile (a quarter of the exponentials are a polynomial's)."""
    Sk, Sq = 400, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k = torch.zeros(1, Sq, 1, D, device=DEV), torch.zeros(1, Sk, 1, D, device=DEV)
    q[..., 0] = 1
    k[..., 0] = -95 * torch.rand(1, Sk, 1, device=DEV, generator=g)
    k[0, :40, 0, 0] = torch.linspace(-1, 0, 40, device=DEV)
    q, k = q.bfloat16().requires_grad_(), k.bfloat16().requires_grad_()
    v = torch.randn(1, Sk, 1, D, device=DEV, generator=g).bfloat16().requires_grad_()
    dout = torch.eye(Sq, D, device=DEV).view(1, Sq, 1, D).bfloat16()
    out = sliding_window_attention(q, k, v, window=Sk, scale=1.0)
    dv = torch.autograd.grad(out, (q, k, v), dout)[2][0, :, 0, :Sq].double()
    _lib.fetch_status()
    seen = build_window_mask(Sq, Sk, Sk, 0, None, DEV)[0]
    want = k.detach()[0, :, 0, 0].double().expand(Sq, Sk).masked_fill(~seen, -math.inf).softmax(-1).t()
    assert (want[want > 0].min() < 2.0 ** -126) and want.max() > 0.02
    # rounded to bf16, and over the sum of the forward's rounded weights; fp32's argument of the exponential (up to 140) is off by 2^-17
    assert ((dv - want).abs() <= (2.1 * U + 2.0 ** -12) * want + 2.0 ** -126).all()
