"""Scratch memory of the sliding-window backward, which packed training asks for at every layer. CPU (the host side of the library)."""
import pytest

from maltos_b200.ops import _lib


@pytest.mark.parametrize("B,S,Hq,Hkv,window,sinks", [(1, 4093, 20, 20, 512, 4), (4, 8192, 32, 8, 1024, 4), (4, 8192, 32, 32, 512, 4), (1, 8192, 32, 8, 1024, 4),
                                                     (1, 131072, 32, 8, 1024, 4), (2, 16384, 8, 2, 4096, 16), (4, 8192, 32, 8, 128, 1000),
                                                     (1, 1024, 8, 8, 256, 4), (8, 2048, 8, 1, 64, 1), (64, 500, 4, 4, 100, 7)])
@pytest.mark.parametrize("D", [64, 128])
def test_scratch_is_no_more_than_the_gradients(B, S, Hq, Hkv, window, sinks, D):
    words = _lib.lib().mb_window_attn_bwd_scratch_words
    gradients = 2 * B * S * Hkv * D * 2                       # dK and dV, bf16
    rows = 2 * B * Hq * ((S + 127) // 128 * 128) * 4           # lse and delta of whole tiles, fp32
    packed, plain = (4 * words(B, S, S, Hq, Hkv, D, window, sinks, p) for p in (1, 0))
    # beside them: the list of work, and what few heads take so that every SM has pieces (148 x 4 pieces of 128 x D, twice, in fp32)
    few = 148 * 4 * 2 * 128 * D * 4 + 2 ** 20
    assert rows < packed <= gradients + rows + few and rows < plain <= gradients + rows + few
    assert 4 * words(B, S, S, Hq, Hkv, D, window, 0, 1) <= rows + few      # no first tokens: no block is cut for them
