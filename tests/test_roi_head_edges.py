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
