"""The serving kernels against plain 64-bit forms: MXFP8 cache, attention over pages, sampling."""
import pytest
import torch

from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.ops import ref

import serving_util as U

pytestmark = pytest.mark.gpu


def _status():
    ops.cuda_module().check_status()


def _rows(seed, B, T, KV, D, spread=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, KV, D, generator=g)
    if spread:     # every magnitude that bf16 has
        x = x * torch.exp2(torch.randint(-130, 127, (B, T, KV, D // 32, 1), generator=g).float()).expand(B, T, KV, D // 32, 32).reshape(x.shape)
    return x.to(torch.bfloat16).cuda()


def _pools(P, page, KV, D):
    k = torch.full((P, page, KV, D), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((P, KV, page, D // 32), 0xA5, dtype=torch.uint8, device="cuda")
    return k, k.clone(), s, s.clone()


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("B,T,KV,D,page", [(1, 1, 1, 64, 16), (5, 37, 3, 128, 16), (2, 130, 10, 128, 8), (64, 1, 10, 128, 16),
                                           (3, 21, 13, 64, 5), (1, 500, 2, 64, 128)])
def test_append_and_read_back(B, T, KV, D, page):
    pages = -(-(T + 40) // page)
    pools = _pools(B * pages + 2, page, KV, D)
    want = [p.clone() for p in pools]
    k, v = _rows(1, B, T, KV, D), _rows(2, B, T, KV, D, spread=True)
    k[0, 0, 0, :32] = 0
    k[-1, -1, -1, -32:] = torch.tensor([448.0, -449.0] * 16)
    table = torch.randperm(B * pages + 2, generator=torch.Generator().manual_seed(3))[: B * pages].to(torch.int32).view(B, pages).cuda()
    pos = (torch.arange(T)[None] + torch.randint(0, 40, (B, 1))).to(torch.int32)
    pos[:, T // 2] = -1
    pos = pos.cuda()
    ops.kv_append_mx(*pools, table, pos, k, v)
    ref.kv_append_mx(*want, table, pos, k, v)
    for a, b in zip(pools, want):           # untouched places hold what they held
        assert torch.equal(a, b)
    got = ops.kv_read_mx(*pools, table, pos)
    for x, y in zip((k, v), got):
        value, _ = U.quantise(x)
        value[pos < 0] = 0
        assert y.dtype == torch.bfloat16 and torch.equal(y, value.to(torch.bfloat16))
    _status()


def test_append_from_strided_rows_and_special_values():
    B, T, KV, D = 2, 9, 4, 128
    pools, want = _pools(4, 16, KV, D), _pools(4, 16, KV, D)
    wide = _rows(5, B, T, 3 * KV, D)
    wide[0, 1, KV, 5], wide[0, 2, KV, 40], wide[1, 0, 2 * KV, 127] = float("nan"), float("inf"), float("-inf")
    wide[1, 3, KV] = 3.0e38
    wide[1, 4, KV] = 1.0e-40
    k, v = wide[:, :, KV:2 * KV], wide[:, :, 2 * KV:]
    odd = torch.zeros(B, T, KV, D + 4, dtype=torch.bfloat16, device="cuda")[..., 4:]      # no 16-byte alignment: copied
    odd.copy_(v)
    table = torch.tensor([[0, 1], [3, 2]], dtype=torch.int32, device="cuda")
    pos = torch.arange(10, 10 + T, dtype=torch.int32, device="cuda")[None].repeat(B, 1)
    ops.kv_append_mx(*pools, table, pos, k, odd)
    ref.kv_append_mx(*want, table, pos, k, v)
    for a, b in zip(pools, want):
        assert torch.equal(a, b)
    ka, va = ops.kv_read_mx(*pools, table, pos)
    kr, vr = ref.kv_read_mx(*want, table, pos)
    for a, b in ((ka, kr), (va, vr)):       # below 2^-126 bf16 itself loses bits: 2^-133 is its last step
        same = (a == b) | (a.isnan() & b.isnan()) | ((a.double() - b.double()).abs() <= 2.0 ** -133)
        assert bool(same.all())
    assert bool(ka[0, 1, 0, :32].isnan().all()) and not bool(ka[0, 1, 0, 32:].isnan().any())
    _status()


def test_append_and_read_leave_bad_places_alone_and_record_them():
    KV, D = 2, 64
    pools = _pools(3, 16, KV, D)
    before = [p.clone() for p in pools]
    table = torch.tensor([[7, -1]], dtype=torch.int32, device="cuda")        # a page outside the pool, an unmapped one
    k = _rows(1, 1, 3, KV, D)
    for at in (3, 20, 40):                                                   # 40: past the table
        pos = torch.tensor([[-1, at, -5]], dtype=torch.int32, device="cuda")
        ops.kv_append_mx(*pools, table, pos, k, k)
        with pytest.raises(RuntimeError, match="outside its table"):
            _status()
        ka, va = ops.kv_read_mx(*pools, table, pos)
        with pytest.raises(RuntimeError, match="outside its table"):
            _status()
        assert not ka.any() and not va.any()
    assert all(torch.equal(a, b) for a, b in zip(pools, before))
    _status()


# ------------------------------------------------------------------------------------------------ attention
def _run(c, window, decode=False, scale=None):
    if decode:
        out = ops.paged_decode_attention_mx(c["q"][:, 0], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], window,
                                            scale)[:, None]
    else:
        out = ops.paged_chunk_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["q_lens"], window, scale,
                                        c["ks"], c["vs"])
    return out


def _variants(c, window, scale):
    """The outputs of both kernels, where both take the call."""
    K = ops.cuda_module()
    for v in (1, 2) if c["k"].shape[1] % 16 == 0 and (scale is None or scale > 0) else (1,):
        yield K.paged_chunk_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["q_lens"], window, scale, c["ks"], c["vs"], v)


def _hold(c, window, decode=False, scale=None):
    out = _run(c, window, decode, scale)
    assert out.shape == c["q"].shape and out.is_contiguous()
    want, bound = U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"], c["lens"],
                              c["q_lens"], window, scale)
    off = (out.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float((off - bound).max()), bad.nonzero()[0].tolist())
    assert torch.equal(out, _run(c, window, decode, scale))          # the same bits again
    if not decode:
        for other in _variants(c, window, scale):
            assert bool(((other.double() - want).abs() <= bound).all())
    _status()


@pytest.mark.parametrize("H,KV,D", [(1, 1, 64), (10, 10, 128), (10, 5, 128), (8, 2, 64), (8, 1, 128), (12, 1, 128), (40, 2, 64),
                                    (6, 2, 128)])
@pytest.mark.parametrize("window", [-1, 0, 17, 300])
def test_decode_mx(H, KV, D, window):
    lens = [1, 0, 2, 15, 16, 17, 100, 333, 1025]
    _hold(U.paged_case(H + D, len(lens), 1, H, KV, D, 16, lens, device="cuda"), window, decode=True)


@pytest.mark.parametrize("page", [1, 7, 8, 32, 48, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_mx_page_sizes(page, D):
    lens = [1, 3, 200, 131]
    _hold(U.paged_case(page, 4, 1, 4, 2, D, page, lens, device="cuda"), -1, decode=True)
    _hold(U.paged_case(page, 4, 1, 4, 2, D, page, lens, device="cuda"), 50, decode=True)


def test_decode_mx_long_and_many():
    _hold(U.paged_case(1, 1, 1, 2, 1, 128, 16, [20000], device="cuda"), -1, decode=True)
    _hold(U.paged_case(2, 70, 1, 5, 5, 64, 16, [(i * 37) % 400 for i in range(70)], device="cuda"), -1, decode=True)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("H,KV,D,page,window", [(10, 10, 128, 16, -1), (10, 5, 128, 16, 100), (4, 2, 64, 16, 37), (6, 2, 128, 8, -1),
                                                (3, 1, 64, 32, 0), (16, 1, 128, 16, -1), (5, 5, 64, 7, 64)])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 40, 130])
def test_chunk(mx, H, KV, D, page, window, T):
    new = [T, 0, 1, max(1, T // 2), T, T]
    past = [0, 50, 300, 17, 129, 1]
    lens = [a + b for a, b in zip(new, past)]
    _hold(U.paged_case(T + D, 6, T, H, KV, D, page, lens, new, mx=mx, device="cuda"), window)


@pytest.mark.parametrize("mx", [False, True])
def test_chunk_without_q_lens_and_with_strides(mx):
    c = U.paged_case(4, 3, 9, 4, 4, 128, 16, [9, 40, 500], mx=mx, device="cuda", stride_pad=24)
    _hold(c, -1)
    _hold(c, -1, scale=0.3)
    c["q"] = c["q"].transpose(1, 2).contiguous().transpose(1, 2)          # heads outside tokens
    _hold(c, 12)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T,H,KV,D,lens,window", [(600, 4, 2, 128, [600, 700], -1), (257, 2, 1, 64, [3000, 257], 500),
                                                  (1000, 2, 2, 128, [1000, 1001], 256)])
def test_long_chunk(mx, T, H, KV, D, lens, window):
    new = [T, T - 3]
    _hold(U.paged_case(T, 2, T, H, KV, D, 16, lens, new, mx=mx, device="cuda"), window)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T", [1, 3, 150])
def test_more_new_tokens_than_the_sequence_has(mx, T):
    """seq_lens below q_lens: the rows before position 0 see nothing and are zero."""
    c = U.paged_case(9, 3, T, 4, 2, 128, 16, [T, 5, 1], None, mx=mx, device="cuda")
    c["lens"] = torch.tensor([T - 1, min(max(T - 2, 0), 5), 0], dtype=torch.int32, device="cuda")
    _hold(c, -1)
    assert not _run(c, -1)[2].any()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T", [1, 70])
def test_unusable_pages_are_left_out_and_recorded(mx, T):
    c = U.paged_case(11, 2, T, 4, 2, 64, 16, [200, 180], mx=mx, device="cuda")
    c["table"][0, 2], c["table"][1, 4] = 10 ** 6, -1
    out = _run(c, -1)
    with pytest.raises(RuntimeError, match="outside its table"):
        _status()
    want, bound = U.attention(c["q"], U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"]), c["table"], c["lens"], None, -1)
    for o in [out, *_variants(c, -1, None)]:
        assert bool(((o.double() - want).abs() <= bound).all())
    ops.cuda_module()._C.reset_status(0)
    c["table"] = c["table"][:, :5].contiguous()         # a table shorter than the sequence
    c["table"][0, 2], c["table"][1, 4] = 0, 0
    c["lens"] = torch.tensor([200, 90], dtype=torch.int32, device="cuda")
    out = _run(c, -1)
    with pytest.raises(RuntimeError, match="outside its table"):
        _status()
    assert out.shape == c["q"].shape
    _status()


@pytest.mark.parametrize("mx", [False, True])
def test_attention_on_another_stream_and_in_graphs(mx):
    """Two captured graphs and eager calls in between, on streams of their own: each has its own workspace."""
    c = [U.paged_case(s, 2, 3, 4, 2, 128, 16, [700, 1500], [3, 2], mx=mx, device="cuda") for s in (1, 2)]
    want = [_run(x, -1) for x in c]
    many = next(iter(list(_variants(c[0], -1, None))[1:]))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert torch.equal(many, list(_variants(c[0], -1, None))[1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in c:
        with torch.cuda.stream(side):
            _run(x, -1)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(x, -1))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager = _run(c[0], -1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    _status()


@pytest.mark.parametrize("T,H,page,scale,why", [(1 << 22, 1, 8, None, "so many new tokens"), (1 << 22, 1, 16, -1.0, "so many new tokens"),
                                                (1 << 22, 1, 16, 0.0, "so many new tokens"), (1 << 24, 1, 16, None, "too large"),
                                                (1 << 20, 1024, 16, None, "too large")])
def test_chunks_too_long_are_refused(T, H, page, scale, why):
    """Nothing is allocated for them: q is broadcast."""
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(1, T, H, 64)
    k = torch.zeros(2, page, 1, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match=why):
        ops.paged_chunk_attention(q, k, k.clone(), table, lens, lens, -1, scale)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
@pytest.mark.parametrize("T", [1, 90])
def test_scales_that_are_not_positive(mx, scale, T):
    _hold(U.paged_case(21, 2, T, 4, 2, 64, 16, [T + 600, T + 3], [T, max(1, T - 2)], mx=mx, device="cuda"), -1, scale=scale)


@pytest.mark.parametrize("mx", [False, True])
def test_two_calls_at_once(mx):
    """Calls on two streams, in flight together, of both kernels: the results are those of calls one after the other."""
    c = [U.paged_case(s, 4, 64, 4, 2, 128, 16, [2000, 700, 64, 1500], [64, 3, 64, 50], mx=mx, device="cuda") for s in (1, 2)]
    want = [list(_variants(x, -1, None)) for x in c]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(list(_variants(c[i], -1, None)))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))
    _status()


def _views(t):
    """The numbers of t in dense rows at an odd address, broadcast along the first dimension, and with an odd stride of a
    dimension of one."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    odd = flat[1:].view(t.shape)
    odd.copy_(t)
    yield odd
    yield t[:1].expand(t.shape)
    one = t[:1].contiguous()
    yield torch.as_strided(one, one.shape, (5, *one.stride()[1:]))


@pytest.mark.parametrize("mx", [False, True])
def test_rows_at_any_address(mx):
    c = U.paged_case(6, 2, 40, 4, 2, 128, 16, [90, 300], [40, 33], mx=mx, device="cuda")
    for q in _views(c["q"]):
        B = q.shape[0]
        part = dict(c, q=q, table=c["table"][:B].contiguous(), lens=c["lens"][:B], q_lens=c["q_lens"][:B])
        for a, b in zip(_variants(part, -1, None), _variants(dict(part, q=q.clone(memory_format=torch.contiguous_format)), -1, None)):
            assert torch.equal(a, b)
    _status()


def test_append_of_rows_at_any_address():
    k = _rows(3, 2, 5, 2, 128).cuda()
    table = torch.arange(2, dtype=torch.int32, device="cuda")[:, None].contiguous()
    for view in _views(k):
        B = view.shape[0]
        pos = torch.arange(5, dtype=torch.int32, device="cuda").repeat(B, 1)
        got = []
        for x in (view, view.clone(memory_format=torch.contiguous_format)):
            pools = [torch.zeros(2, 16, 2, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
            pools += [torch.zeros(2, 2, 16, 4, dtype=torch.uint8, device="cuda") for _ in range(2)]
            ops.kv_append_mx(*pools, table[:B].contiguous(), pos, x, x)
            got.append(pools)
        assert all(torch.equal(a, b) for a, b in zip(*got))
    _status()


# ------------------------------------------------------------------------------------------------ sampling
def _logits(seed, R, V, bf16, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(R, V, generator=g) * scale).to(torch.bfloat16)
    z[:, : max(1, V // 50)] += 4
    return z.cuda() if bf16 else (15 * torch.tanh(z.float() / 15)).cuda(), torch.rand(R, generator=g).cuda()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 33), (4, 1000), (3, 4097), (2, 50257), (2, 65536), (1, 131072)])
@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 0.99, 0.0), (1.0, 2000, 0.95, 0.0),
                                     (1.0, 0, 1.0, 0.1), (0.9, 40, 0.8, 0.02), (0.0, 0, 1.0, 0.0), (5.0, 5000, 0.97, 0.001),
                                     (1.0, 1, 0.5, 0.0), (1.0, 3, 0.0, 0.0), (0.01, 0, 0.9999, 0.0)])
def test_sample_rows(bf16, R, V, t, k, p, m):
    z, u = _logits(V + k, R, V, bf16)
    got = ops.sample_rows(z, u, t, k, p, m)
    assert got.dtype == torch.int64 and torch.equal(got.cpu(), U.sample(z, u, t, k, p, m))


@pytest.mark.parametrize("bf16", [False, True])
def test_sample_rows_with_settings_of_their_own(bf16):
    R, V = 60, 3001
    z, u = _logits(8, R, V, bf16)
    g = torch.Generator().manual_seed(1)
    pick = lambda xs: [xs[int(i)] for i in torch.randint(0, len(xs), (R,), generator=g)]  # noqa: E731
    t, k, p, m = pick([0.0, 0.5, 1.0, 2.0]), pick([0, 1, 7, 1500]), pick([1.0, 0.9, 0.4]), pick([0.0, 0.05, 1.0])
    c = lambda x, d: torch.tensor(x, dtype=d).cuda()  # noqa: E731
    got = ops.sample_rows(z, u, c(t, torch.float32), c(k, torch.int32), c(p, torch.float32), c(m, torch.float32))
    assert torch.equal(got.cpu(), U.sample(z, u, t, k, p, m))
    got = ops.sample_rows(z, u, c(t, torch.float32), 20, c(p, torch.float32), 0.0)
    assert torch.equal(got.cpu(), U.sample(z, u, t, 20, p, 0.0))


@pytest.mark.parametrize("setting", [(1.0, 0, 1.0, 0.0), (1.0, 100, 1.0, 0.0), (1.0, 1500, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 2500, 0.5, 0.0),
                                     (1.0, 0, 1.0, 1.0), (0.5, 2000, 0.3, 0.5), (0.0, 0, 1.0, 0.0)])
def test_sample_rows_ties_and_masks(setting):
    V = 3000
    rows = [torch.zeros(V),                                              # all equal
            torch.full((V,), float("-inf")).index_fill(0, torch.tensor([5, 77, 2998]), 1.0),
            torch.full((V,), torch.finfo(torch.float32).min).index_fill(0, torch.tensor([9]), 0.0),
            torch.full((V,), torch.finfo(torch.float32).min),            # nothing but the type's lowest value
            torch.full((V,), float("-inf")), torch.full((V,), float("nan")),
            torch.cat([torch.tensor([float("nan"), float("inf"), 3.0, float("inf")]), torch.zeros(V - 4)]),
            torch.cat([torch.zeros(V // 2), torch.ones(V - V // 2)]),
            (torch.arange(V) % 7).float(), torch.cat([torch.tensor([-0.0]), torch.zeros(V - 1)]),
            1.0e30 * torch.arange(V).float(), 1.0e-42 * torch.arange(V).float()]
    z = torch.stack(rows).cuda()
    for u0 in (0.0, 0.25, 0.61803, 0.9999999):
        u = torch.full((len(rows),), u0, device="cuda")
        got, want = ops.sample_rows(z, u, *setting).cpu(), U.sample(z, u, *setting)
        assert torch.equal(got, want), (u0, got.tolist(), want.tolist())


def test_sample_rows_from_strided_logits_and_edges():
    z, u = _logits(3, 7, 1000, True)
    wide = torch.full((7, 1061), 100.0, dtype=torch.bfloat16, device="cuda")
    for off in (0, 1, 3, 8):                     # rows that start anywhere: what lies beside them is not read
        part = wide[:, off:off + 1000]
        part.copy_(z)
        assert torch.equal(ops.sample_rows(part, u, 1.0, 0, 0.9).cpu(), U.sample(z, u, 1.0, 0, 0.9, 0.0))
        wide.fill_(100.0)
    assert ops.sample_rows(z[:0], u[:0]).shape == (0,)
    one = torch.ones(7, device="cuda")           # outside [0, 1): taken as its ends
    assert torch.equal(ops.sample_rows(z, one * 2).cpu(), ops.sample_rows(z, one).cpu())
    assert torch.equal(ops.sample_rows(z, -one).cpu(), ops.sample_rows(z, one * 0).cpu())


def test_sample_rows_captured():
    z, u = _logits(4, 16, 5000, False)
    ops.sample_rows(z, u, 1.0, 50, 0.9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.sample_rows(z, u, 1.0, 50, 0.9)
    for seed in (5, 6):
        z2, u2 = _logits(seed, 16, 5000, False)
        z.copy_(z2), u.copy_(u2)
        g.replay()
        assert torch.equal(out.cpu(), U.sample(z2, u2, 1.0, 50, 0.9, 0.0))


# ------------------------------------------------------------------------------------------------ together
def test_append_attend_sample_together():
    """A prompt chunk and then single tokens: quantise and write, attend over what was written, sample a token."""
    B, T, H, KV, D, page, pages = 3, 21, 4, 2, 128, 16, 4
    g = torch.Generator().manual_seed(0)
    pools = _pools(B * pages, page, KV, D)
    table = torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages).cuda()
    head = torch.randn(H * D, 500, generator=g).to(torch.bfloat16).cuda()
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    stored = None
    for step, n in enumerate((T, 1, 1, 4)):
        q, k, v = (_rows(10 * step + i, B, n, h, D) for i, h in ((0, H), (1, KV), (2, KV)))
        pos = (lens[:, None] + torch.arange(n, dtype=torch.int32, device="cuda")[None]).contiguous()
        ops.kv_append_mx(*pools, table, pos, k, v)
        lens = lens + n
        new = [U.quantise(x)[0] for x in (k, v)]
        stored = new if stored is None else [torch.cat([a, b], 1) for a, b in zip(stored, new)]
        if n == 1:
            out = ops.paged_decode_attention_mx(q[:, 0], *pools, table, lens)[:, None]
        else:
            out = ops.paged_chunk_attention(q, pools[0], pools[1], table, lens, k_scale=pools[2], v_scale=pools[3])
        flat = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]        # the same rows as one page a sequence
        want, bound = U.attention(q, stored[0], stored[1], flat, lens, None, -1)
        assert bool(((out.double() - want).abs() <= bound).all())
        logits = out[:, -1].reshape(B, -1).float() @ head.float()
        u = torch.rand(B, generator=g).cuda()
        assert torch.equal(ops.sample_rows(logits, u, 0.9, 40, 0.9).cpu(), U.sample(logits, u, 0.9, 40, 0.9, 0.0))
    _status()


def test_refusals():
    """The same refusals as on the CPU, and tensors on different devices."""
    import test_serving_ops_cpu as C
    C.refusals_of_the_cache("cuda")
    C.refusals_of_attention("cuda")
    C.refusals_of_sampling("cuda")
    for name in ("v_pool", "k_scale", "page_table", "positions", "k_new"):
        a = C._cache_args("cuda")
        a[name] = a[name].cpu()
        with pytest.raises(RuntimeError):
            ops.kv_append_mx(**a)
    with pytest.raises(RuntimeError):
        ops.sample_rows(torch.zeros(2, 8, device="cuda"), torch.zeros(2))
