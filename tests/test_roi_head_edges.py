"""The RoI head's operators where sizes meet the kernels' own limits: an axis of one, counts under long padding, walks that are not
split, many images, long sums.  Values and bounds come from the definitions in 64 bits in test_roi_head.  Where roi_attention_backward
gets the forward's `rest`, delta is formed from the output before its rounding, so that its own error is 2^-16 of its terms."""
import math

import pytest
import torch

from test_roi_head import _attn64, _attn_inputs, _close, _gen


# ------------------------------------------------------------------ an axis of one
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Nq,Nk", [(1, 70), (70, 1), (1, 1)])
def test_roi_attention_one_row_of_a_far_apart_bank(Nq, Nk, dtype):
    """One row, or one key, of a bank whose rows lie farther apart than 32 bits of bytes hold: an axis of one has no stride, and the
    call gives the bits of the dense one."""
    from vision_amd import ops
    B, H, D = 3, 2, 128
    dense = [t.cuda() for t in _attn_inputs(61, B, Nq, Nk, H, H, D, dtype)]
    q, k, v, do = dense
    out, lse = ops.roi_attention(q, k, v)
    grads = ops.roi_attention_backward(do, q, k, v, out, lse)
    for far in ((1 << 22) + 64, 1 << 26, 1 << 31, (1 << 40) + 192):
        views = []
        for t in dense:
            if t.shape[1] != 1:
                views.append(t)
                continue
            wide = torch.zeros((B, 3, H, D), dtype=dtype, device="cuda")           # heads of one of three fused tensors: not dense
            wide[:, 1] = t[:, 0]
            views.append(wide.as_strided((B, 1, H, D), (3 * H * D, far, D, 1), H * D))
        a, b, c, g = views
        o, s = ops.roi_attention(a, b, c)
        assert torch.equal(o, out) and torch.equal(s, lse), far
        assert all(torch.equal(x, y) for x, y in zip(ops.roi_attention_backward(g, a, b, c, out, lse), grads)), far


# ------------------------------------------------------------------ few keys under long padding
@pytest.mark.gpu
@pytest.mark.parametrize("Nk", [700, 2000])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_roi_attention_gradient_of_few_counted_keys(D, Nk):
    """Images padded to more keys than those for which ds is cut in two by size alone: the count decides.  1, 3 and 7 keys of equal score:
    p is 1 / n, the sum of ds over them 0, and dq, the sum of ds k over equal k, 0 too.  delta comes from out and its rest, 2^-16 of
    |do| |out| apart, ds goes into its products as two parts, 2^-16 of it, and 32-bit sums of D terms add D 2^-24 of their
    magnitudes.  The fourth image has all its keys, at the usual bounds."""
    from vision_amd import fast_rcnn
    N, u2, E32, counts = 150, 2.0 ** -16, 2.0 ** -24, (1, 3, 7, Nk)
    q, k, v, do = _attn_inputs(81, 4, N, Nk, 2, 1, D, torch.bfloat16)
    k[:3] = k[:3, :1]
    kc = torch.tensor(counts).int()
    want = _attn64(q[3:], k[3:], v[3:], None, None, None, None, do[3:])
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(fast_rcnn.roi_attention(*leaves, k_counts=kc.cuda()), leaves, do.cuda())
    q, k, v, do = (t.double() for t in (q, k, v, do))
    for b, n in enumerate(counts[:3]):
        V = v[b, :n, 0]
        o = V.mean(0)
        dp = do[b] @ V.T                             # (N, 2, n)
        at = (do[b].abs() @ o.abs())[..., None]
        ds = (dp - (do[b] @ o)[..., None]) / n
        mag = do[b].abs() @ V.abs().T + at
        eds = ds.abs() * (u2 + 16 * E32) + (at * u2 + (D + 8) * E32 * mag) / n + 8 * E32 * dp.abs() / n
        sc = D ** -0.5
        edq = (eds + n * E32 * ds.abs()).sum(-1, keepdim=True) * k[b, 0, 0].abs() * sc
        _close(dq[b], (torch.zeros_like(q[b]), edq), ("dq", n))
        wdk = torch.einsum("ihj,ihd->jd", ds, q[b]) * sc
        edk = torch.einsum("ihj,ihd->jd", eds + 2 * N * E32 * ds.abs(), q[b].abs()) * sc + 2.0 ** -8 * wdk.abs()
        _close(dk[b, :n, 0], (wdk, edk), ("dk", n))
        assert float(dk[b, n:].abs().max()) == 0.0 and float(dv[b, n:].abs().max()) == 0.0
    for got, name in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        _close(got[3:], want[name], name)


# ------------------------------------------------------------------ long sums
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("above", [0.3, 1.0, 1.7])
def test_roi_attention_long_sum_of_equal_scores(above, dtype):
    """16001 keys of equal score behind a first one `above` them, enough rows that the walk is not split: the roundings of a sum of equal
    terms do not average out.  lse: the terms share one relative error, of the score's product (3 units of 2^-24 of it: the query's value is
    exact, scale, maximum and the rounding of the exponent's argument), and of the exponential (2); a tile's sum adds 5 levels, the
    compensated sum over the tiles 4 and the two lanes 1; the logarithm 2 units of its value.  out, of equal values, is 1: numerator and
    denominator each hold those errors, and the numerator's sum, which the matrix cores add up by 16 keys, at most 12 roundings a tile of 32
    keys; at the end a division and the rounding to the type."""
    from vision_amd import ops
    B, N, M, H, D, E32 = 1, 4096, 16001, 8, 8, 2.0 ** -24
    q, k = torch.zeros((B, N, H, D), dtype=dtype), torch.zeros((B, M, H, D), dtype=dtype)
    q[..., 0] = 1.0
    k[:, 0, :, 0] = above
    v = torch.ones((B, M, H, D), dtype=dtype)
    out, lse = ops.roi_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
    s = float(k[0, 0, 0, 0])
    want = math.log(math.exp(s) + (M - 1))
    el = (3 * s + 2 + 5 + 4 + 1) * E32
    err = float((lse.cpu().double() - want).abs().max())
    assert err <= el + 2 * E32 * want, err / E32
    eo = 12 * (M // 32 + 1) * E32 + 2 * el + 2 * E32 + (2.0 ** -8 + 2.0 ** -8 if dtype == torch.bfloat16 else E32)
    assert float((out.cpu().double() - 1.0).abs().max()) <= eo


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,c", [(4096, 131072), (300, 1000003), (300, 131072), (1, 131072)])
def test_class_logprobs_long_sum_of_equal_scores(n, c, dtype):
    """1024 equal scores before many equal lower ones, so that every lane's sum starts from a maximum above the rest.  The terms share one
    relative error, of the exponent's argument (its size) and of the exponential (2 units of 2^-24); a turn's sum of sixteen adds 16,
    sixteen turns 16, the sums put away one each (a wave alone takes 16384 scores for one, four waves four times as many), lanes,
    waves and splits at most 8 joins of 2; log probabilities add 2 units of the logarithm's and their own size, the entropy as much of its
    two terms."""
    from vision_amd import ops
    E32 = 2.0 ** -24
    for above in (0.3, 1.0, 1.7):
        z = torch.zeros((n, c), dtype=dtype, device="cuda")
        z[:, :1024] = above
        s = float(z[0, 0])
        y = torch.arange(n, device="cuda") % 2 * (c - 1)                      # the first class or the last
        logp, entropy, _, _, _ = ops.class_logprobs(z, y)
        del z
        L = math.log(1024 * math.exp(s) + c - 1024)
        H = -(1024 * math.exp(s - L) * (s - L) - (c - 1024) * math.exp(-L) * L)
        es = (s + 2 + 16 + 16 + c / 16384 + 16) * E32
        want = torch.where(y == 0, s - L, -L).double()
        assert float(((logp.double() - want).abs() - (es + 2 * E32 * (L - s + want.abs()))).max()) <= 0.0, above
        spread = (c - 1024) * math.exp(-L) * s                                # w / s of the kernel's formula
        assert float((entropy.double() - H).abs().max()) <= es + 2 * E32 * (L - s) + spread * (2 * es + 4 * E32) + E32 * H, above


# ------------------------------------------------------------------ refusals
def test_rest_of_float32_is_refused():
    """On the host, before any launch: rest is of bf16, and a DG_F32 call that took it would clear padded rows at twice its size."""
    import ctypes as C
    from vision_amd import _abi
    lib = _abi.load()
    s = _abi.AttnShape(1, 8, 8, 1, 1, 64)
    for t in "qkvg":
        for a, n in (("batch", 512), ("row", 64), ("head", 64)):
            setattr(s, f"{t}_stride_{a}", n)
    s.scale, s.dtype = 0.125, _abi.F32
    p = C.c_void_p(4096)                         # never touched: the calls end before a launch
    assert lib.dg_roi_attn_fwd(s, p, p, p, None, None, None, p, p, p, p, 1 << 30, None) == _abi.EINVAL
    assert "rest" in _abi.last_error()
    assert lib.dg_roi_attn_bwd(s, p, p, p, p, p, p, p, None, None, None, p, p, p, p, 1 << 30, None) == _abi.EINVAL
    assert "rest" in _abi.last_error()


# ------------------------------------------------------------------ walks that are not split, many images
def _both(case, dtype, seed, qc, kc, mask=None):
    from vision_amd import ops
    q, k, v, do = _attn_inputs(seed, *case, dtype)
    want = _attn64(q, k, v, qc, kc, mask, None, do)
    Q, K, V, G, QC, KC, M = (None if t is None else t.cuda() for t in (q, k, v, do, qc, kc, mask))
    out, lse, rest = ops.roi_attention(Q, K, V, QC, KC, M, rest=True)
    _close(out, want["out"], "out")
    _close(lse, want["lse"], "lse")
    for name, got in zip(("dq", "dk", "dv"), ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M, rest=rest)):
        _close(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(32, torch.bfloat16), (64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
@pytest.mark.parametrize("ragged", [False, True])
def test_roi_attention_walks_that_are_not_split(D, dtype, ragged):
    """256 tiles of rows and of keys and more: every workgroup walks all of its image, the maximum is renewed on the way, images and
    heads go round the compute dies; ragged: one image of few keys, one of few rows, one of all."""
    q, k = (torch.tensor([1900, 130, 1333]).int(), torch.tensor([300, 1900, 1200]).int()) if ragged else (None, None)
    _both((3, 1900, 1900, 6, 6, D), dtype, 71, q, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("masked", [False, True])
def test_roi_attention_many_images(masked, dtype):
    """More images than a wave has lanes, which are taken in their own order; some without rows or keys."""
    g = _gen(73)
    B, Nq, Nk = 70, 45, 150
    q, k = torch.randint(0, Nq + 1, (B,), generator=g).int(), torch.randint(0, Nk + 1, (B,), generator=g).int()
    _both((B, Nq, Nk, 4, 2, 40), dtype, 72, q, k, torch.rand((B, Nq, Nk), generator=g) < 0.4 if masked else None)


@pytest.mark.gpu
def test_heads_of_no_size_are_refused():
    from vision_amd import fast_rcnn, ops
    q, k = torch.zeros((1, 3, 2, 0), device="cuda"), torch.zeros((1, 4, 2, 0), device="cuda")
    for call in (lambda: ops.roi_attention(q, k, k), lambda: fast_rcnn.roi_attention(q, k, k)):
        with pytest.raises(ValueError, match="head size"):
            call()
