"""Drop-ins for rcnn/fast_rcnn.py.

  slowroipool(output_size).foward(img, roi_ary, roi_idx)   rcnn/fast_rcnn.py:351-377
  nms(rects, scores) -> (rect, score)                      rcnn/fast_rcnn.py:590-610

and, with no counterpart there (its sketch classifies every RoI by itself, :379-384), what a head that relates the RoIs of an
image to each other trains on, with gradients:

  roi_attention(q, k, v, ...)                              attention over an image's RoIs or map cells
  rope_axes(q, k, pos, plan)                               rotary positions from box centres, frames, rows and columns
  class_logprobs(logits, labels, top)                      log probabilities of the labels, entropy, best classes

As written the reference pools with AdaptiveAvgPool2d stored in a field called `maxpool`
(:354) and never defines backward (autograd).  `mode="avg"` (the default: an import swap must
reproduce the class as written) is that; `mode="max"` is the RoI MAX-pooling north_star asks
for -- the same module with AdaptiveMaxPool2d substituted -- and also yields the argmax used
by the backward scatter.
"""
from collections import namedtuple

import numpy as np
import torch

from . import ops


class _RoIPoolFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, img, win, mode, size):
        small = tuple(size) == (7, 7) and img.shape[2] * img.shape[3] <= 65535
        out, argmax = ops.roipool_forward(img, win, mode, P=size,
                                          argmax_dtype=torch.int16 if small else torch.int32)   # uint16 indices: half the bytes
        ctx.mode, ctx.img_shape, ctx.size = mode, tuple(img.shape), tuple(size)
        ctx.save_for_backward(win, argmax if argmax is not None else win)
        ctx.argmax = argmax
        return out

    @staticmethod
    def backward(ctx, grad_out):
        win, arg = ctx.saved_tensors
        g = ops.roipool_backward(grad_out.contiguous(), arg if ctx.mode == "max" else None, win, ctx.img_shape, ctx.mode, P=ctx.size)
        return g, None, None, None


class slowroipool(torch.nn.Module):
    def __init__(self, output_size, mode="avg"):
        super().__init__()
        size = tuple(int(v) for v in output_size) if isinstance(output_size, (tuple, list)) else (int(output_size), int(output_size))
        if len(size) != 2 or min(size) < 1:
            raise ValueError("slowroipool: output_size must be a positive int or a pair of them")
        if mode not in ("max", "avg"):
            raise ValueError("mode must be 'max' or 'avg'")
        self.size = size
        self.mode = mode
        self.argmax = None            # (n,C,PH,PW) int32 of the last max-mode forward (flat y*W+x in the map)

    def foward(self, img, roi_ary, roi_idx):          # sic: the reference's spelling (:357)
        was_cpu = not img.is_cuda
        dev = ops._abi.device_of(img)
        x = img.to(device=dev, dtype=torch.float32)
        B, C, H, W = x.shape
        win, status = ops.roi_windows(np.asarray(roi_ary, np.float64) if not isinstance(roi_ary, torch.Tensor) else roi_ary,
                                      np.asarray(roi_idx, np.int64) if not isinstance(roi_idx, torch.Tensor) else roi_idx,
                                      B, H, W, dev)
        st = int(status.item())
        if st & 1:
            raise RuntimeError("slowroipool: a RoI crop is empty (x2<=x1 or y2<=y1 after floor/ceil)")
        if st & 2:
            raise IndexError("slowroipool: roi_idx out of range")
        if x.requires_grad:
            out = _RoIPoolFn.apply(x, win, self.mode, self.size)
        else:
            out, self.argmax = ops.roipool_forward(x, win, self.mode, P=self.size)
        return out.cpu() if was_cpu else out

    forward = foward


def nms(rects, scores):
    """rcnn/fast_rcnn.py:590-610.  The reference's function of this name does no suppression: it orders the rects by
    np.argsort(scores)[::-1] and returns element 0 -- the rect of the maximal score, taken on the scores as given
    (float64).  That is what runs here (dg_top_score_f64): exact on scores that differ below fp32 resolution; equal
    maxima resolve to the highest index (in the reference the order among equal keys is whatever numpy's unstable
    argsort produces, so its pick among exactly tied scores is implementation-defined)."""
    rects_a = np.array(rects)
    scores_a = np.array(scores)
    if scores_a.size == 0:
        raise IndexError("index 0 is out of bounds for axis 0 with size 0")     # what nms_rects[0] raises in the reference
    dev = ops._abi.device_of(None)
    sc = ops._abi.to_dev(scores_a.astype(np.float64).reshape(-1), torch.float64, dev)
    top = torch.empty((1,), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        ops.check(ops.load().dg_top_score_f64(ops.ptr(sc), sc.shape[0], ops.ptr(top), ops.stream_ptr(dev)))
    top = int(top.item())
    return rects_a[top], scores_a[top]


# ------------------------------------------------------------------ RoI head
def _once(backward):
    """torch's once_differentiable, without its cost where no graph of the gradient is asked for"""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return call


class _RoIAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_counts, k_counts, mask, scale):
        args = ops._attn_args(q, k, v, q_counts, k_counts, mask)
        out, lse, rest = ops._attn_forward(args, scale, any(ctx.needs_input_grad))
        ctx.save_for_backward(*args[1:7], out, lse, rest)     # as they were laid out for the kernels
        ctx.rest = args[0], args[7], args[8], scale
        return out

    @staticmethod
    @_once
    def backward(ctx, grad_out):
        *args, out, lse, rest = ctx.saved_tensors
        dev, masks, ms, scale = ctx.rest
        need = ctx.needs_input_grad
        dq, dk, dv = ops._attn_backward((dev, *args, masks, ms), grad_out, out, lse, rest, scale, need[0], need[1] or need[2])
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def roi_attention(q, k, v, q_counts=None, k_counts=None, mask=None, scale=None):
    """ops.roi_attention's out, with a gradient for q, k and v.  Tensors on the CPU are copied in and the result back."""
    dev = ops._abi.device_of(q, k, v)
    was_cpu = not (q.is_cuda or k.is_cuda or v.is_cuda)
    if not (q.device == dev and k.device == dev and v.device == dev):
        q, k, v = q.to(dev), k.to(dev), v.to(dev)
    if mask is not None and not isinstance(mask, torch.Tensor):
        mask = torch.as_tensor(mask)
    out = _RoIAttentionFn.apply(q, k, v, q_counts, k_counts, mask, scale)
    return out.cpu() if was_cpu else out


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, plan, inverse):
        args = ops._rope_args(q, k, pos, plan)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(args[3])
        ctx.rest = args[0], args[4], inverse
        return ops._rope_turn(*args, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        (pos,) = ctx.saved_tensors
        dev, plan, inverse = ctx.rest
        if dq is None and dk is None:
            return None, None, None, None, None
        g, h = dk[:, :, :0] if dq is None else dq, dq[:, :, :0] if dk is None else dk
        g, h = _RopeFn.apply(g, h, pos, plan, not inverse) if torch.is_grad_enabled() else ops._rope_turn(dev, g, h, pos, plan, not inverse)
        return None if dq is None else g, None if dk is None else h, None, None, None


def rope_axes(q, k, pos, plan):
    """ops.rope_axes of queries and keys in one launch, with a gradient for both (none for the positions).  Tensors on the CPU
    are copied in and the results back."""
    dev = ops._abi.device_of(q, k)
    was_cpu = not (q.is_cuda or k.is_cuda)
    if not isinstance(pos, torch.Tensor) or pos.device != dev:
        pos = torch.as_tensor(pos, device=dev)
    if pos.requires_grad:
        raise ValueError("rope_axes: positions have no gradient here; detach them")
    if not (q.device == dev and k.device == dev):
        q, k = q.to(dev), k.to(dev)
    q, k = _RopeFn.apply(q, k, pos, plan, False)
    return (q.cpu(), k.cpu()) if was_cpu else (q, k)


class _ClassLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top):
        dev, z, y = ops._logits(logits, labels, "class_logprobs")
        logp, entropy, norm, best, index = ops._logprobs(dev, z, y, top)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(z, y, norm, entropy)
        ctx.mark_non_differentiable(best, index)
        return logp, entropy, best, index

    @staticmethod
    @_once
    def backward(ctx, g, gh, _best, _index):
        z, y, norm, entropy = ctx.saved_tensors
        if g is None and gh is None:
            return None, None, None
        g, gh = (t if t is None else t.contiguous() for t in (g, gh))
        return ops._logprobs_backward(z.device, z, y, norm, entropy, g, gh), None, None


ClassLogprobs = namedtuple("ClassLogprobs", "logp entropy top_logp top_index")


def class_logprobs(logits, labels=None, top=0):
    """ops.class_logprobs' logp, entropy, top_logp and top_index, with a gradient of logp and entropy for the logits: the loss of
    a classifier of RoIs is -logp.sum() / n over the labelled rows (label_proposals' labels; a negative label is left out).
    Tensors on the CPU are copied in and the results back."""
    dev = ops._abi.device_of(logits)
    was_cpu = not logits.is_cuda
    r = _ClassLogprobsFn.apply(logits.to(dev) if was_cpu else logits, labels, int(top))
    return ClassLogprobs(*(t if t is None else t.cpu() for t in r)) if was_cpu else ClassLogprobs(*r)
