"""The few-rows attention kernel where its runs of keys are long, and the memory that a call takes."""
import pytest
import torch

from nanochat_cpp_b200 import ops

import serving_util as U

pytestmark = pytest.mark.gpu


def _peak(fn):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = fn()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("window", [-1, 2000])
def test_workspace_does_not_grow_with_rows_times_table(mx, window):
    """Many rows and a wide table, on pages that only this kernel takes: besides the output no more than half a gigabyte."""
    B, T, H, KV, D, page = 8, 2048, 32, 8, 128, 8
    table = torch.full((B, 2304), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(B)
    k = torch.zeros(B, page, KV, D, dtype=torch.uint8 if mx else torch.bfloat16, device="cuda")
    s = torch.full((B, KV, page, D // 32), 127, dtype=torch.uint8, device="cuda") if mx else None
    q = torch.zeros(B, T, H, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.full((B,), 8, dtype=torch.int32, device="cuda")
    new = torch.full((B,), 5, dtype=torch.int32, device="cuda")
    out, peak = _peak(lambda: ops.paged_chunk_attention(q, k, k, table.cuda(), lens, new, window, None, s, s))
    assert peak - out.numel() * 2 - table.numel() * 4 < (1 << 29) and not out.any()
    ops.cuda_module().check_status()


@pytest.mark.parametrize("H,KV,T", [(8, 8, 1), (10, 10, 13), (32, 4, 4), (6, 2, 50)])
@pytest.mark.parametrize("window", [-1, 2000])
def test_workspace_is_bounded_for_any_number_of_units(H, KV, T, window):
    """Under 7104 units there are at most twice as many runs and two more per unit: 28416 runs of 32 rows of D + 2 numbers."""
    for B in (1, 33, 200):
        table = torch.full((B, 65536), -1, dtype=torch.int32, device="cuda")
        k = torch.zeros(1, 8, KV, 64, dtype=torch.bfloat16, device="cuda")
        q = torch.zeros(B, T, H, 64, dtype=torch.bfloat16, device="cuda")
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        out, peak = _peak(lambda: ops.paged_chunk_attention(q, k, k, table, lens, None, window))
        assert peak <= 28416 * 32 * (64 + 2) * 4 + out.numel() * 2 + 4096 and not out.any()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("page,window", [(16, -1), (32, 900), (48, -1), (128, -1), (7, -1), (16, 1200)])
def test_long_runs(mx, page, window):
    """A table so much wider than the sequences that a run is a whole sequence of more than 512 keys."""
    T, width = 1300, 400000
    new = [T, T - 60]
    c = U.paged_case(page, 2, T, 4, 4, 64, page, [1600, 1301], new, mx=mx, device="cuda")
    table = torch.full((2, -(-width // page)), -1, dtype=torch.int32, device="cuda")
    table[:, :c["table"].shape[1]] = c["table"]
    K = ops.cuda_module()
    out = K.paged_chunk_attention(c["q"], c["k"], c["v"], table, c["lens"], c["q_lens"], window, None, c["ks"], c["vs"], 1)
    want, bound = U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"], c["lens"],
                              c["q_lens"], window)
    assert bool(((out.double() - want).abs() <= bound).all())
    K.check_status()
    bad = table.clone()
    bad[0, 1100 // page] = 10 ** 6             # one page behind the first 512 keys
    out = K.paged_chunk_attention(c["q"], c["k"], c["v"], bad, c["lens"], c["q_lens"], window, None, c["ks"], c["vs"], 1)
    with pytest.raises(RuntimeError, match="outside its table"):
        K.check_status()
    want, bound = U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), bad, c["lens"],
                              c["q_lens"], window)
    assert bool(((out.double() - want).abs() <= bound).all())
