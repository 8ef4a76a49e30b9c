"""Attention over the pages: tables shorter than their sequences, and one prompt cut into pieces."""
import pytest
import torch

from nanochat_cpp_b200 import ops

import serving_range_util as R
import serving_util as U

pytestmark = pytest.mark.gpu


def _want(c, window=-1):
    return U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"], c["lens"], c["q_lens"], window)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T,window", [(1, -1), (70, -1), (70, 20), (150, 100)])
def test_keys_past_the_table_are_left_out(mx, T, window):
    """Five pages of sequences of 200 and 130 tokens: the keys of those pages alone count, and rows whose window lies behind them
    are zero. Both kernels, and the status word."""
    c = U.paged_case(31, 2, T, 4, 2, 64, 16, [200, 130], mx=mx, device="cuda")
    c["table"] = c["table"][:, :5].contiguous()
    want, bound = _want(c, window)
    calls = [lambda v=v: R.run(c, v, window) for v in (0, R.ROWS, R.CHUNK)]
    if mx and T == 1:
        calls.append(lambda: ops.paged_decode_attention_mx(c["q"][:, 0], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], window)[:, None])
    for call in calls:
        out = call()
        assert bool(((out.double() - want).abs() <= bound).all())
        if window >= 0:
            first = 200 - T                        # position of row 0; keys end at 80
            assert not out[0, max(0, 80 + window - first):].any()
        with pytest.raises(RuntimeError, match="outside its table"):
            ops.cuda_module().check_status()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("D,window", [(128, -1), (64, 200)])
def test_one_prompt_in_pieces(mx, D, window):
    """The rows of a prompt, whole (by size the many-rows kernel) and in pieces (the few-rows one, and both): each within the bound
    of its own roundings, so two cuts differ by twice that at most."""
    B, T, H, KV = 2, 640, 16, 8
    c = U.paged_case(5, B, T, H, KV, D, 16, [T, T], mx=mx, device="cuda")
    want, bound = _want(c, window)
    for piece in (T, 1, 7, 100, 333):
        if piece == 1:
            starts = range(0, T, 61)
        else:
            starts = range(0, T, piece)
        for s in starts:
            n = min(piece, T - s)
            lens = torch.full((B,), s + n, dtype=torch.int32, device="cuda")
            out = ops.paged_chunk_attention(c["q"][:, s:s + n], c["k"], c["v"], c["table"], lens, None, window, None, c["ks"], c["vs"])
            assert bool(((out.double() - want[:, s:s + n]).abs() <= bound[:, s:s + n]).all())
    ops.cuda_module().check_status()
