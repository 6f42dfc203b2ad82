"""The RoI head's operators against their definitions in 64 bits: attention over an image's boxes (forward, backward), rotary
positions over several axes, log probabilities of labels.

Tolerances.  One rounding to a type moves a value by at most half a step, u = 2^-8 of it in bf16, 2^-11 in fp16, 2^-24 in fp32.
Attention in bf16: p (and ds) is rounded once as an operand, the result once at the end, so an output element is off by at most
u sum |p_ij v_j| + u |o_i|, and the sum itself is held in 32 bits; delta is formed from the rounded out (u |do| |out| per row).
Each bound below is such a sum of magnitudes, formed in 64 bits from the same inputs, plus the 32-bit terms: a product of d
terms is off by at most d 2^-24 sum |q k| scale, which moves p by that factor."""
import math

import numpy as np
import pytest
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E32 = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _attn64(q, k, v, qc, kc, mask, scale, do=None):
    """definition in 64 bits on the CPU, with the bounds of the module's text: dict of (value, bound)"""
    u = 2.0 ** -24 if q.dtype == torch.float32 else 2.0 ** -8
    B, Nq, Hq, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)     # noqa: E731
    out, lse, dq, dk, dv = z(B, Nq, Hq, D), torch.full((B, Hq, Nq), -math.inf, dtype=torch.float64), z(B, Nq, Hq, D), z(B, Nk, Hk, D), z(B, Nk, Hk, D)
    tout, tlse, tdq, tdk, tdv = z(B, Nq, Hq, D), z(B, Hq, Nq), z(B, Nq, Hq, D), z(B, Nk, Hk, D), z(B, Nk, Hk, D)
    for b in range(B):
        n = Nq if qc is None else min(max(int(qc[b]), 0), Nq)
        m = Nk if kc is None else min(max(int(kc[b]), 0), Nk)
        see = torch.ones(n, m, dtype=torch.bool) if mask is None else mask[b if mask.shape[0] > 1 else 0, :n, :m].bool()
        for h in range(Hq):
            j = h // (Hq // Hk)
            Q, K, V = q[b, :n, h].double(), k[b, :m, j].double(), v[b, :m, j].double()
            s = (Q @ K.T) * scale
            s = torch.where(see, s, torch.full_like(s, -math.inf))
            L = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64)
            p = torch.where(see, torch.exp(s - torch.where(torch.isinf(L), torch.zeros_like(L), L)[:, None]), torch.zeros_like(s))
            # relative error of a probability in 32 bits: the product's, the exponent's argument and its statistic, the exponential
            ep = (D + 4) * E32 * (Q.abs() @ K.abs().T) * scale + 8 * E32 * (1 + torch.where(torch.isinf(L), torch.zeros_like(L), L.abs())[:, None]) + \
                8 * E32 * torch.where(see, s.abs(), torch.zeros_like(s)) + m * E32
            o = p @ V
            out[b, :n, h], lse[b, h, :n] = o, L
            eo = (p * (2 * ep + u)) @ V.abs() + u * o.abs()
            tout[b, :n, h] = eo
            tlse[b, h, :n] = torch.where(torch.isinf(L), torch.zeros_like(L), (p * ep).sum(1) + 4 * E32 * (1 + L.abs()))
            if do is not None:
                G = do[b, :n, h].double()
                dp = G @ V.T
                delta = (G * o).sum(1, keepdim=True)
                edp = (D + 4) * E32 * (G.abs() @ V.abs().T) + (G.abs() * eo).sum(1, keepdim=True) + (D + 4) * E32 * (G.abs() * o.abs()).sum(1, keepdim=True)
                ds = p * (dp - delta)
                eds = ds.abs() * (2 * ep + u + 2 * E32) + p * edp
                dv[b, :m, j] += p.T @ G
                tdv[b, :m, j] += (p * (2 * ep + u + n * E32)).T @ G.abs()
                dq[b, :n, h] = ds @ K * scale
                tdq[b, :n, h] = (eds + m * E32 * ds.abs()) @ K.abs() * scale + u * (ds @ K * scale).abs()
                dk[b, :m, j] += ds.T @ Q * scale
                tdk[b, :m, j] += (eds + n * (Hq // Hk) * E32 * ds.abs()).T @ Q.abs() * scale
    tdk += u * dk.abs()
    tdv += u * dv.abs()
    r = dict(out=(out, tout), lse=(lse, tlse))
    if do is not None:
        r.update(dq=(dq, tdq), dk=(dk, tdk), dv=(dv, tdv))
    return r


def _close(got, want, what):
    w, tol = want
    g = got.detach().cpu().double()
    assert g.shape == w.shape, what
    same = (g == w) | (torch.isnan(g) & torch.isnan(w))
    off = torch.where(same, torch.zeros_like(w), (g - w).abs() - (tol + 1e-30))
    assert not torch.isnan(off).any(), (what, "NaN")
    assert float(off.max() if off.numel() else 0.0) <= 0.0, (what, float(off.max()), int((off > 0).sum()), float((g - w).abs().max()))


def _attn_inputs(seed, B, Nq, Nk, Hq, Hk, D, dtype):
    g = _gen(seed)
    q, k, v, do = (torch.randn(s, generator=g).to(dtype) for s in ((B, Nq, Hq, D), (B, Nk, Hk, D), (B, Nk, Hk, D), (B, Nq, Hq, D)))
    return q, k, v, do


ATTN_CASES = [
    # B, Nq, Nk, Hq, Hk, D, counts, mask
    (1, 1, 1, 1, 1, 8, False, None),
    (1, 1, 5000, 8, 2, 128, False, None),        # one query, split over the keys
    (2, 1, 700, 4, 4, 64, True, None),
    (1, 3, 1, 2, 1, 32, False, None),
    (2, 33, 65, 2, 2, 40, False, None),
    (1, 128, 64, 1, 1, 64, False, None),
    (2, 129, 127, 6, 2, 64, True, None),
    (3, 98, 98, 4, 4, 32, True, "pairs"),
    (2, 200, 257, 4, 1, 128, True, "pairs"),
    (1, 5000, 40, 2, 2, 64, False, None),        # few keys, many rows: dk, dv split over the rows
    (1, 700, 900, 2, 2, 72, False, "shared"),
    (2, 64, 100, 2, 1, 104, True, "none"),       # a mask that leaves every row empty
    (4, 50, 50, 3, 3, 16, "zero", None),         # images with no rows or no keys at all
]


def _attn_masks(case, seed):
    B, Nq, Nk, Hq, Hk, D, counts, mask = case
    g = _gen(seed + 1)
    qc = kc = None
    if counts:
        qc, kc = torch.randint(0, Nq + 1, (B,), generator=g).int(), torch.randint(0, Nk + 1, (B,), generator=g).int()
        qc[0], kc[0] = max(1, Nq - 1), max(1, Nk - 1)
        if counts == "zero":
            qc[1], kc[2], kc[3] = 0, 0, Nk + 5
        else:
            qc[-1] = max(1, int(qc[-1]))
    m = None
    if mask == "pairs":
        m = (torch.rand((B, Nq, Nk), generator=g) < 0.3) & (torch.rand((B, Nq, 1), generator=g) > 0.1)
    elif mask == "shared":
        m = (torch.rand((1, Nq, Nk), generator=g) < 0.5)
    elif mask == "none":
        m = torch.zeros((B, Nq, Nk), dtype=torch.bool)
    return qc, kc, m


def _dev(t):
    return None if t is None else t.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", ATTN_CASES, ids=lambda c: "x".join(map(str, c)))
def test_roi_attention(case, dtype):
    from vision_amd import ops
    q, k, v, do = _attn_inputs(7, *case[:6], dtype)
    qc, kc, m = _attn_masks(case, 7)
    want = _attn64(q, k, v, qc, kc, m, None, do)
    if qc is not None:                           # what lies behind a count is never read
        for b in range(case[0]):
            q[b, max(int(qc[b]), 0):] = math.nan
            do[b, max(int(qc[b]), 0):] = math.inf
            k[b, max(int(kc[b]), 0):] = math.nan
            v[b, max(int(kc[b]), 0):] = math.inf
    Q, K, V, G, QC, KC, M = map(_dev, (q, k, v, do, qc, kc, m))
    out, lse = ops.roi_attention(Q, K, V, QC, KC, M)
    _close(out, want["out"], "out")
    _close(lse, want["lse"], "lse")
    dq, dk, dv = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M)
    _close(dq, want["dq"], "dq")
    _close(dk, want["dk"], "dk")
    _close(dv, want["dv"], "dv")
    out2, lse2 = ops.roi_attention(Q, K, V, QC, KC, M)             # the same bits in every run
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    again = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))
    only_q = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M, need_kv=False)
    only_kv = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M, need_q=False)
    assert torch.equal(only_q[0], dq) and only_q[1] is None and only_kv[0] is None
    assert torch.equal(only_kv[1], dk) and torch.equal(only_kv[2], dv)
