"""Sliding-window attention where its ordinary cases do not reach. Oracle and bounds: test_window_attention_gpu."""
import math

import pytest
import torch

from maltos_b200.ops import _lib
from maltos_b200.ops.attention import sliding_window_attention, sliding_window_reference
from tests.test_window_attention_gpu import DEV, _expect, _qkv

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
