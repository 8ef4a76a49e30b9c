"""Attention cases whose numbers span what the cache formats hold, with an error bound that follows each score."""
import torch

import serving_util as U
from nanochat_cpp_b200 import ops
from nanochat_cpp_b200.ops import ref

PAGE = 16
ROWS, CHUNK = 1, 2      # the two kernels of paged_chunk_attention


def case(q, k, v, lens, mx, q_lens=None, page=PAGE, width=None):
    """q [B, T, H, D], k / v [B, S, KV, D] (numbers that bf16 holds): pools with the rows of sequence b on pages of its own, of
    which `width` (default: as many as needed) are in the table."""
    B, S, KV, D = k.shape
    pages = -(-S // page)
    c = dict(q=q.to(torch.bfloat16).cuda(), ks=None, vs=None, lens=torch.tensor(lens, dtype=torch.int32).cuda(),
             q_lens=None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32).cuda())
    table = torch.arange(B * pages, dtype=torch.int32).flip(0).view(B, pages)
    c["table"] = torch.full((B, max(width or 0, pages)), -1, dtype=torch.int32)
    c["table"][:, :pages] = table
    c["table"] = c["table"].cuda()
    for n, x in (("k", k), ("v", v)):
        rows = torch.zeros(B, pages * page, KV, D, dtype=torch.bfloat16)
        rows[:, :S] = x.to(torch.bfloat16)
        pool = torch.zeros(B * pages, page, KV, D, dtype=torch.bfloat16)
        pool[table.long().view(-1)] = rows.view(B * pages, page, KV, D)
        if mx:
            pool, scale = ref.mx_kv_encode(pool)
            c[n + "s"] = scale.permute(0, 2, 1, 3).contiguous().cuda()
        c[n] = pool.contiguous().cuda()
    return c


def expect(c, window=-1, scale=None, exact_products=False, score_error=None):
    """(result, bound) in 64 bits. As in `serving_util.attention`, with u = 2^-8 for a rounding to bf16 and A = sum w_j |v_j|:
    rounding the probabilities moves the quotient by u (A + |o|), rounding the result by u |o|. An error d_j of score j, however,
    counts with its own weight: sum_j w_j d_j (|v_j| + |o|), so that a key of enormous size and no weight does not
    loosen the bound. d_j = (D + 2) 2^-24 |scale| sum |q_i k_ji| + 2^-21 for fp32 sums of products and the exponential; where all
    products and sums are whole numbers below 2^24 only the scaling rounds: 4 * 2^-24 |s_j| + 2^-21. 1 % for second order. Below 2^-126
    bf16 steps by 2^-133: half a step for the values and half for the result are added. `score_error`: another d_j."""
    q, B, T, H, D = c["q"].double(), *c["q"].shape
    k, v = U.pool_values(c["k"], c["ks"]), U.pool_values(c["v"], c["vs"])
    KV, page = k.shape[2], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    u = 2.0 ** -8
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        L, n = int(c["lens"][b]), T if c["q_lens"] is None else int(c["q_lens"][b])
        S = min(L, c["table"].shape[1] * page)
        j = torch.arange(S, device=q.device)
        if S <= 0:
            continue
        pg = c["table"][b].long()[j // page]
        kk, vv = k[pg, j % page], v[pg, j % page]
        at = torch.arange(L - n, L, device=q.device)[:, None]
        seen = (j[None] <= at) & ((at - j[None] <= window) if window >= 0 else (j[None] >= 0))
        some = seen.any(1)
        for h in range(H):
            g = h // (H // KV)
            qh, kh, vh = q[b, :n, h], kk[:, g], vv[:, g]
            s = qh @ kh.T * scale
            w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            w = torch.where(some[:, None], w, torch.zeros_like(w))
            if score_error is not None:
                d = torch.full_like(s, score_error)
            elif exact_products:
                d = 4 * 2.0 ** -24 * s.abs() + 2.0 ** -21
            else:
                d = (D + 2) * 2.0 ** -24 * (qh.abs() @ kh.abs().T) * abs(scale) + 2.0 ** -21
            o, A = w @ vh, w @ vh.abs()
            wd = torch.where(w > 0, w * d, torch.zeros_like(w))
            out[b, :n, h] = o
            bound[b, :n, h] = 1.01 * (u * A + 2 * u * o.abs() + wd @ vh.abs() + wd.sum(-1, keepdim=True) * o.abs()) + 2.0 ** -133
    return out, bound


def unit(g, *shape):
    x = torch.randn(*shape, generator=g)
    return x * 1.2 / x.square().mean(-1, keepdim=True).sqrt()


def run(c, variant, window=-1, scale=None):
    return ops.cuda_module().paged_chunk_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["q_lens"], window, scale,
                                                   c["ks"], c["vs"], variant)


def hold(c, variant, window=-1, scale=None, exact_products=False, score_error=None):
    out = run(c, variant, window, scale)
    want, bound = expect(c, window, scale, exact_products, score_error)
    bad = ~((out.double() - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), float(out[bad][0]), float(want[bad][0]))
    ops.cuda_module().check_status()
