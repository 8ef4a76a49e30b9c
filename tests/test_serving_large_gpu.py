"""The serving kernels over pools beyond 4 GB, and the many-rows kernel in a graph."""
import pytest
import torch

from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.ops import ref

import serving_range_util as R
import serving_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", [R.ROWS, R.CHUNK])
@pytest.mark.parametrize("mx", [False, True])
def test_pages_behind_four_gigabytes(variant, mx):
    """A small case moved to the last pages of a large pool: the same bits. The pool's bytes and elements pass 32 bits."""
    c = U.paged_case(1, 2, 40, 4, 4, 128, 16, [300, 77], [40, 33], mx=mx, device="cuda")
    want = R.run(c, variant)
    n = c["k"].shape[0]
    row = 16 * 4 * 128                                   # elements of a page
    pages = (9 << 29) // row if mx else (5 << 29) // row   # 4.8e9 bytes; 2.7e9 elements, 5.4e9 bytes
    big = dict(c, table=torch.where(c["table"] >= 0, c["table"] + (pages - n), c["table"]))
    for name in ("k", "v", "ks", "vs") if mx else ("k", "v"):
        pool = torch.empty(pages, *c[name].shape[1:], dtype=c[name].dtype, device="cuda")
        pool[:n] = 0x7F if mx else float("nan")          # where a wrapped offset would read
        pool[pages - n:] = c[name]
        big[name] = pool
    assert torch.equal(R.run(big, variant), want)
    ops.cuda_module().check_status()


def test_append_behind_four_gigabytes():
    KV, D, page = 4, 128, 16
    pages = (9 << 29) // (page * KV * D)
    codes = [torch.empty(pages, page, KV, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, KV, page, D // 32, dtype=torch.uint8, device="cuda") for _ in range(2)]
    k, v = (torch.randn(2, 30, KV, D, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 4], [pages - 2, pages - 3]], dtype=torch.int32, device="cuda")
    pos = torch.arange(30, dtype=torch.int32, device="cuda").repeat(2, 1)
    ops.kv_append_mx(*codes, *scales, table, pos, k, v)
    got = ops.kv_read_mx(*codes, *scales, table, pos)
    for x, y in zip((k, v), got):
        assert torch.equal(y, U.quantise(x)[0].to(torch.bfloat16))
    first, eb = ref.mx_kv_encode(k[0, :16])
    assert torch.equal(codes[0][-1], first) and torch.equal(scales[0][-1], eb.permute(1, 0, 2))
    ops.cuda_module().check_status()


@pytest.mark.parametrize("mx", [False, True])
def test_the_many_rows_kernel_in_two_graphs(mx):
    """Captured with key runs and their workspace; replayed in turn, with other lengths and numbers in the same tensors."""
    c = [U.paged_case(s, 2, 40, 4, 2, 128, 16, [1500, 2000], [40, 40], mx=mx, device="cuda") for s in (1, 2)]
    graphs, outs = [], []
    for x in c:
        R.run(x, R.CHUNK)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(R.run(x, R.CHUNK))
        graphs.append(g)
    for step in range(3):
        want = [R.run(x, R.CHUNK) for x in c]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        for x in c:
            x["q"].copy_(x["q"].flip(1))
            x["lens"].sub_(torch.tensor([301, 64 * step], dtype=torch.int32, device="cuda"))
            x["q_lens"].copy_(torch.tensor([40 - 7 * step, step], dtype=torch.int32, device="cuda"))
    ops.cuda_module().check_status()
