"""Tensor-level front end of the HIP kernels: GPU tensors in, GPU tensors out, async on the
current stream.  The reference-named drop-ins (yolo_v1.py, yolo_v2.py, rcnn_utils.py,
fast_rcnn.py, cluster.py) are thin layers over these."""
import functools
import math

import torch

from . import _abi
from ._abi import check, load, ptr, stream_ptr, workspace


def _f32c(t, dev):
    return _abi.to_dev(t, torch.float32, dev)


# ------------------------------------------------------------------ IoU
def iou_elementwise(bb1, bb2, eps=1e-7):
    dev = _abi.device_of(bb1, bb2)
    f64 = isinstance(bb1, torch.Tensor) and bb1.dtype == torch.float64
    dt = torch.float64 if f64 else torch.float32
    a, b = _abi.to_dev(bb1, dt, dev).reshape(-1, 4), _abi.to_dev(bb2, dt, dev).reshape(-1, 4)
    if a.shape != b.shape:
        raise ValueError(f"get_iou: shapes differ {tuple(a.shape)} vs {tuple(b.shape)}")
    out = torch.empty(a.shape[0], dtype=dt, device=dev)
    fn = load().dg_iou_elementwise_f64 if f64 else load().dg_iou_elementwise_f32
    with torch.cuda.device(dev):
        check(fn(ptr(a), ptr(b), a.shape[0], eps, ptr(out), stream_ptr(dev)))
    return out


def iou_pairwise(a, b, eps=1e-7, out=None):
    dev = _abi.device_of(a, b)
    a, b = _f32c(a, dev).reshape(-1, 4), _f32c(b, dev).reshape(-1, 4)
    if out is None:
        out = torch.empty((a.shape[0], b.shape[0]), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        check(load().dg_iou_pairwise_f32(ptr(a), a.shape[0], ptr(b), b.shape[0], eps, ptr(out), stream_ptr(dev)))
    return out


def iou_rois_vs_gt(rois, grt):
    """float64 IoU of n xyxy rois against one box + per-roi assert flags (rcnn/utils.py:50-67)."""
    dev = _abi.device_of(rois, grt)
    r = _abi.to_dev(rois, torch.float64, dev).reshape(-1, 4)
    g = _abi.to_dev(grt, torch.float64, dev).reshape(4)
    out = torch.empty(r.shape[0], dtype=torch.float64, device=dev)
    flags = torch.empty(r.shape[0], dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        check(load().dg_iou_rois_vs_gt_f64(ptr(r), ptr(g), r.shape[0], ptr(out), ptr(flags), stream_ptr(dev)))
    return out, flags


# ------------------------------------------------------------------ NMS
def nms_workspace(dev, batch, nmax):
    nbytes = load().dg_nms_workspace_bytes(batch, nmax)
    return workspace(dev, nbytes), nbytes


def nms_path_info(dev, batch, nmax, img=0):
    """(mode, fpdone, rounds, npairs, cand_per_box, est_pairs_per_box) of image `img` in the LAST NMS call that used this
    stream's workspace: mode 0 = pruned pair search, 1 = dense mask; fpdone 1 = the fixed-point kernel produced the keep list.
    Synchronous (diagnostic)."""
    import ctypes as C
    ws, nbytes = nms_workspace(dev, batch, nmax)
    out = (C.c_int32 * 6)()
    with torch.cuda.device(dev):
        check(load().dg_nms_path_info(ptr(ws), nbytes, batch, nmax, img, out))
    return tuple(out)


def nms_batched(boxes, scores, counts=None, threshold=0.1, quirk_drop_last=True, keep=None, keep_count=None):
    """boxes (B,N,4) fp32, scores (B,N), counts (B) int32 or None -> keep (B,N) int64, keep_count (B) int32."""
    dev = _abi.device_of(boxes, scores)
    boxes, scores = _f32c(boxes, dev), _f32c(scores, dev)
    B, N = scores.shape
    if boxes.shape != (B, N, 4):
        raise ValueError("nms_batched: boxes must be (B,N,4) matching scores (B,N)")
    if counts is not None:
        counts = _abi.to_dev(counts, torch.int32, dev)
    if keep is None:
        keep = torch.empty((B, N), dtype=torch.int64, device=dev)
    if keep_count is None:
        keep_count = torch.empty((B,), dtype=torch.int32, device=dev)
    ws, nbytes = nms_workspace(dev, B, N)
    with torch.cuda.device(dev):
        check(load().dg_nms_batched_f32(ptr(boxes), ptr(scores), ptr(counts), B, N, float(threshold), int(quirk_drop_last),
                                        ptr(keep), ptr(keep_count), ptr(ws), nbytes, stream_ptr(dev)))
    return keep, keep_count


def nms_batched_per_class(boxes, scores, labels, num_classes, counts=None, threshold=0.1, quirk_drop_last=True):
    """Per-class NMS (no reference counterpart: its nms is class-agnostic, yolo.py:188-203): the reference's nms applied to
    each class's boxes of an image separately.  labels (B,N) int64 in [0,num_classes).
    -> keep (B,N) int64 (classes' keep lists concatenated in class order), keep_count (B), class_count (B,num_classes)."""
    dev = _abi.device_of(boxes, scores)
    boxes, scores = _f32c(boxes, dev), _f32c(scores, dev)
    labels = _abi.to_dev(labels, torch.int64, dev)
    B, N = scores.shape
    if boxes.shape != (B, N, 4) or labels.shape != (B, N):
        raise ValueError("nms_batched_per_class: boxes (B,N,4), scores (B,N), labels (B,N)")
    if counts is not None:
        counts = _abi.to_dev(counts, torch.int32, dev)
    keep = torch.empty((B, N), dtype=torch.int64, device=dev)
    keep_count = torch.empty((B,), dtype=torch.int32, device=dev)
    class_count = torch.empty((B, int(num_classes)), dtype=torch.int32, device=dev)
    status = torch.zeros((1,), dtype=torch.int32, device=dev)
    nbytes = load().dg_nms_per_class_workspace_bytes(B, N, int(num_classes))
    ws = workspace(dev, nbytes)
    with torch.cuda.device(dev):
        check(load().dg_nms_batched_per_class_f32(ptr(boxes), ptr(scores), ptr(labels), ptr(counts), B, N, int(num_classes),
                                                  float(threshold), int(quirk_drop_last), ptr(keep), ptr(keep_count),
                                                  ptr(class_count), ptr(status), ptr(ws), nbytes, stream_ptr(dev)))
    return keep, keep_count, class_count, status


# ------------------------------------------------------------------ YOLOv1 decode
def yolo1_decode_batched(output, target=None, conf_threshold=0.2, prob_threshold=0.1, nms_threshold=None, per_class=False,
                         quirk_drop_last=True):
    """decode of a batch; with nms_threshold the NMS runs in the same launch (dg_yolo1_decode_nms_f32) and the result
    gains (keep (B,98) int64, keep_count (B) int32, class_count (B,C) int32)."""
    dev = _abi.device_of(output, target)
    o = _f32c(output, dev)
    if o.dim() == 3:
        o = o.unsqueeze(0)
    B = o.shape[0]
    if tuple(o.shape[1:3]) != (7, 7) or o.shape[3] < 11:
        raise ValueError("decode: output must be (...,7,7,10+C)")
    C_ = o.shape[3] - 10
    t = None
    if target is not None:
        t = _f32c(target, dev).reshape(o.shape)
    box = torch.empty((B, 98, 4), dtype=torch.float32, device=dev)
    label = torch.empty((B, 98), dtype=torch.int64, device=dev)
    conf = torch.empty((B, 98), dtype=torch.float32, device=dev)
    score = torch.empty((B, 98), dtype=torch.float32, device=dev)
    count = torch.empty((B,), dtype=torch.int32, device=dev)
    tbox = torch.empty((B, 4), dtype=torch.float64, device=dev) if t is not None else None
    tlabel = torch.empty((B,), dtype=torch.int64, device=dev) if t is not None else None
    if nms_threshold is not None:
        keep = torch.empty((B, 98), dtype=torch.int64, device=dev)
        kcnt = torch.empty((B,), dtype=torch.int32, device=dev)
        ccnt = torch.empty((B, C_), dtype=torch.int32, device=dev) if per_class else None
        with torch.cuda.device(dev):
            check(load().dg_yolo1_decode_nms_f32(ptr(o), ptr(t), B, C_, float(conf_threshold), float(prob_threshold),
                                                 float(nms_threshold), int(bool(per_class)), int(bool(quirk_drop_last)), ptr(box),
                                                 ptr(label), ptr(conf), ptr(score), ptr(count), ptr(keep), ptr(kcnt), ptr(ccnt),
                                                 ptr(tbox), ptr(tlabel), stream_ptr(dev)))
        return box, label, conf, score, count, tbox, tlabel, keep, kcnt, ccnt
    with torch.cuda.device(dev):
        check(load().dg_yolo1_decode_f32(ptr(o), ptr(t), B, C_, float(conf_threshold), float(prob_threshold), ptr(box), ptr(label),
                                         ptr(conf), ptr(score), ptr(count), ptr(tbox), ptr(tlabel), stream_ptr(dev)))
    return box, label, conf, score, count, tbox, tlabel


def yolo1_encode_batched(bb, label, num_classes):
    """bb (n,4) {left, top, w, h}, label (n) in 1..C -> target (n,7,7,10+C) float64 on the GPU (modules.py:151-174)."""
    dev = _abi.device_of(bb, label)
    b = _abi.to_dev(bb, torch.float64, dev).reshape(-1, 4)
    l = _abi.to_dev(label, torch.int64, dev).reshape(-1)
    if l.shape[0] != b.shape[0]:
        raise ValueError("encode: one label per box")
    n = b.shape[0]
    target = torch.empty((n, 7, 7, 10 + num_classes), dtype=torch.float64, device=dev)
    status = torch.zeros((1,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        check(load().dg_yolo1_encode_f64(ptr(b), ptr(l), n, num_classes, ptr(target), ptr(status), stream_ptr(dev)))
    return target, status


# ------------------------------------------------------------------ YOLOv1 loss (fused geometry)
def yolo1_loss(modely, targety, quirk_slot2=True, want_grad=True):
    """(n,7,7,10+C) fp32 x2 -> (loss6 device tensor [loss, xy, wh, obj, noobj, label], grad or None)."""
    dev = _abi.device_of(modely, targety)
    y, t = _f32c(modely, dev), _f32c(targety, dev)
    if y.dim() != 4 or tuple(y.shape[1:3]) != (7, 7) or y.shape[3] < 10 or y.shape != t.shape:
        raise ValueError("Loss: modely/targety must both be (n,7,7,10+C)")
    n, C_ = y.shape[0], y.shape[3] - 10
    loss6 = torch.empty((6,), dtype=torch.float32, device=dev)
    grad = torch.empty_like(y) if want_grad else None
    nbytes = load().dg_yolo1_loss_workspace_bytes(n)
    ws = workspace(dev, nbytes)
    with torch.cuda.device(dev):
        check(load().dg_yolo1_loss_f32(ptr(y), ptr(t), n, C_, int(quirk_slot2), ptr(loss6), ptr(grad), ptr(ws), nbytes, stream_ptr(dev)))
    return loss6, grad


def voc_ap(det_img, det_cls, det_conf, det_box, tgt_img, tgt_cls, tgt_box, num_classes, num_images, iou_thr):
    """VOC-style AP of yolo.py:306-367 for every class in one launch.  Detections and targets are flat device (or host)
    arrays in the reference's list order; returns (ap float64 (C,), n_grt int32 (C,)) on the device.
    The ordering (class, then confidence descending, stable) is two stable torch sorts; the rest is k_voc_ap."""
    dev = _abi.device_of(det_box, tgt_box)
    C_, I = int(num_classes), int(num_images)
    dimg = _abi.to_dev(det_img, torch.int32, dev).reshape(-1)
    dcls = _abi.to_dev(det_cls, torch.int64, dev).reshape(-1)
    dconf = _abi.to_dev(det_conf, torch.float64, dev).reshape(-1)
    dbox = _f32c(det_box, dev).reshape(-1, 4)
    timg = _abi.to_dev(tgt_img, torch.int32, dev).reshape(-1)
    tcls = _abi.to_dev(tgt_cls, torch.int32, dev).reshape(-1)
    tbox = _f32c(tgt_box, dev).reshape(-1, 4)
    n = dimg.shape[0]
    if not (dcls.shape[0] == dconf.shape[0] == dbox.shape[0] == n) or not (timg.shape[0] == tcls.shape[0] == tbox.shape[0]):
        raise ValueError("ap: ragged detection / target arrays")
    if n:
        by_conf = torch.sort(dconf, descending=True, stable=True).indices
        by_cls = torch.sort(dcls[by_conf], stable=True).indices
        order = by_conf[by_cls].to(torch.int32)
        counts = torch.bincount(dcls.clamp(0, C_ - 1), minlength=C_)
    else:
        order = torch.empty(0, dtype=torch.int32, device=dev)
        counts = torch.zeros(C_, dtype=torch.int64, device=dev)
    cls_off = torch.zeros(C_ + 1, dtype=torch.int64, device=dev)
    cls_off[1:] = torch.cumsum(counts, 0)
    out = torch.empty(C_, dtype=torch.float64, device=dev)
    n_grt = torch.empty(C_, dtype=torch.int32, device=dev)
    nbytes = load().dg_voc_ap_workspace_bytes(n, C_, I)
    ws = workspace(dev, nbytes)
    with torch.cuda.device(dev):
        check(load().dg_voc_ap_f32(ptr(dimg), ptr(dbox), ptr(order), ptr(cls_off), n, ptr(timg), ptr(tcls), ptr(tbox),
                                   timg.shape[0], C_, I, float(iou_thr), ptr(out), ptr(n_grt), ptr(ws), nbytes, stream_ptr(dev)))
    return out, n_grt


# ------------------------------------------------------------------ RoI pooling
def roi_windows(rois, roi_idx, B, H, W, dev):
    r = _abi.to_dev(rois, torch.float64, dev).reshape(-1, 4)
    idx = _abi.to_dev(roi_idx, torch.int64, dev).reshape(-1)
    if idx.shape[0] != r.shape[0]:
        raise ValueError("roi_idx must have one entry per RoI")
    win = torch.empty((r.shape[0], 5), dtype=torch.int32, device=dev)
    status = torch.zeros((1,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        check(load().dg_roi_windows(ptr(r), ptr(idx), r.shape[0], B, H, W, ptr(win), ptr(status), stream_ptr(dev)))
    return win, status


def to_nhwc(img, out=None, nan_flag=None):
    """(B,C,H,W) fp32 -> ((B,H,W,C) staging copy, nan_flag).  nan_flag is a device int32 that is non-zero iff
    the map holds a NaN (None for a tensor that already is channels_last: no copy, NaN state unknown)."""
    B, C_, H, W = img.shape
    if img.is_contiguous(memory_format=torch.channels_last) and not img.is_contiguous():
        return img.permute(0, 2, 3, 1), None       # same bytes, viewed NHWC
    img = img.contiguous()
    if out is None:
        out = torch.empty((B, H, W, C_), dtype=torch.float32, device=img.device)
    if nan_flag is None:
        nan_flag = torch.zeros((1,), dtype=torch.int32, device=img.device)
    else:
        nan_flag.zero_()
    with torch.cuda.device(img.device):
        check(load().dg_nchw_to_nhwc_f32(ptr(img), B, C_, H, W, ptr(out), ptr(nan_flag), stream_ptr(img.device)))
    return out, nan_flag


def _pool_size(P):
    if isinstance(P, (tuple, list)):
        if len(P) != 2:
            raise ValueError("output_size must be an int or a (PH, PW) pair")
        return int(P[0]), int(P[1])
    return int(P), int(P)


def roipool_forward(img, win, mode="max", P=7, out=None, argmax=None, nhwc=None, nan_flag=None, argmax_dtype=torch.int32):
    """P: output size, an int or (PH, PW) (rcnn/fast_rcnn.py:352-355 passes it to the adaptive pool).
    argmax: int32 (default) or, with argmax_dtype=torch.int16 / an int16 tensor passed in, the uint16 bit pattern of the
    same index (widen with `argmax_i32`): half the index bytes in the forward and the backward (7 x 7, H*W <= 65535 only)."""
    dev = img.device
    B, C_, H, W = img.shape
    PH, PW = _pool_size(P)
    n = win.shape[0]
    if nhwc is None:
        nhwc, nan_flag = to_nhwc(img)
    m = _abi.POOL_MAX if mode == "max" else _abi.POOL_AVG
    if out is None:
        out = torch.empty((n, C_, PH, PW), dtype=torch.float32, device=dev)
    if m == _abi.POOL_MAX and argmax is None:
        argmax = torch.empty((n, C_, PH, PW), dtype=argmax_dtype, device=dev)
    a16 = m == _abi.POOL_MAX and argmax.dtype == torch.int16
    if m == _abi.POOL_MAX and argmax.dtype not in (torch.int32, torch.int16):
        raise ValueError("roipool_forward: argmax must be int32 or int16 (uint16 bit pattern)")
    with torch.cuda.device(dev):
        if a16:
            if (PH, PW) != (7, 7):
                raise ValueError("roipool_forward: the uint16 argmax exists for 7 x 7 outputs only")
            check(load().dg_roipool_fwd_a16_f32(ptr(nhwc), B, C_, H, W, ptr(win), n, 7, m, ptr(nan_flag), ptr(out), ptr(argmax), stream_ptr(dev)))
        else:
            check(load().dg_roipool_fwd_any_f32(ptr(nhwc), B, C_, H, W, ptr(win), n, PH, PW, m, ptr(nan_flag), ptr(out),
                                                ptr(argmax) if m == _abi.POOL_MAX else None, stream_ptr(dev)))
    return out, (argmax if m == _abi.POOL_MAX else None)


def argmax_i32(argmax):
    """int32 view of an argmax tensor of either width (the 16-bit form holds the uint16 bit pattern)."""
    return argmax if argmax.dtype == torch.int32 else argmax.to(torch.int32) & 0xFFFF


def roipool_backward(grad_out, argmax, win, img_shape, mode="max", P=7, grad_in=None):
    dev = grad_out.device
    B, C_, H, W = img_shape
    PH, PW = _pool_size(P)
    n = win.shape[0]
    g = grad_out.contiguous()
    if grad_in is None:
        grad_in = torch.empty((B, C_, H, W), dtype=torch.float32, device=dev)
    nbytes = load().dg_roipool_bwd_workspace_bytes(B, n)
    ws = workspace(dev, nbytes)
    m = _abi.POOL_MAX if mode == "max" else _abi.POOL_AVG
    with torch.cuda.device(dev):
        if argmax is not None and argmax.dtype == torch.int16:
            check(load().dg_roipool_bwd_a16_f32(ptr(g), ptr(argmax), ptr(win), n, B, C_, H, W, PH, m, ptr(grad_in), ptr(ws), nbytes, stream_ptr(dev)))
        else:
            check(load().dg_roipool_bwd_any_f32(ptr(g), ptr(argmax), ptr(win), n, B, C_, H, W, PH, PW, m, ptr(grad_in), ptr(ws), nbytes,
                                                stream_ptr(dev)))
    return grad_in


# ------------------------------------------------------------------ k-means
def kmeans_step(wh, cent, labels, acc):
    dev = wh.device
    n, k = wh.shape[0], cent.shape[0]
    nbytes = load().dg_kmeans_workspace_bytes(n, k)
    ws = workspace(dev, nbytes)
    with torch.cuda.device(dev):
        check(load().dg_kmeans_iou_step(ptr(wh), n, ptr(cent), k, ptr(labels), ptr(acc), ptr(ws), nbytes, stream_ptr(dev)))
    return acc


def kmeans_run(wh, cent, labels, acc, history, slot0, iters):
    """iters Lloyd iterations on one device without returning to Python in between."""
    dev = wh.device
    n, k = wh.shape[0], cent.shape[0]
    nbytes = load().dg_kmeans_workspace_bytes(n, k)
    ws = workspace(dev, nbytes)
    with torch.cuda.device(dev):
        check(load().dg_kmeans_iou_run(ptr(wh), n, ptr(cent), k, ptr(labels), ptr(acc), ptr(history), slot0, iters, ptr(ws), nbytes,
                                       stream_ptr(dev)))


def kmeans_finish(part, k, cent=None, acc_out=None, history=None, slot=0):
    """fold a partial-sums buffer (all-reduced when sharded): acc_out <- sums, cent moved by them, history[slot] <- changed"""
    dev = part.device
    with torch.cuda.device(dev):
        check(load().dg_kmeans_finish(ptr(part), k, ptr(cent), ptr(acc_out), ptr(history), slot, stream_ptr(dev)))


def kmeans_labels_i32(labels_u8):
    out = torch.empty(labels_u8.shape, dtype=torch.int32, device=labels_u8.device)
    with torch.cuda.device(labels_u8.device):
        check(load().dg_kmeans_labels_i32(ptr(labels_u8), labels_u8.numel(), ptr(out), stream_ptr(labels_u8.device)))
    return out


# ------------------------------------------------------------------ RoI head: attention
def _scratch(nbytes, like):
    """Scratch of one call on a tensor's device, from the caching allocator in the current stream's order: captured graphs and
    calls on other streams never share it."""
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _call(dev, fn, *args):
    """an entry point on its tensors' device, which mostly is the current one"""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args)
    if rc:
        check(rc)


def _empty_like(t):
    """half the time of torch.empty(t.shape, dtype=..., device=...), which a small call spends several times"""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _at(t):
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev):
    """the current stream's handle; through torch.cuda.current_stream it costs 2 us of a call's 15"""
    return _raw_stream(dev.index) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


@functools.lru_cache(maxsize=1024)
def _strides_fit(shape, strides, e):
    """whether a kernel that loads 16 bytes at a time can step along a (B,N,H,D) tensor: a dense last axis, everything else a
    multiple of 16 bytes, rows at most 2^22 values apart"""
    return strides[3] == 1 and all(n == 1 or st * e % 16 == 0 for n, st in zip(shape[:3], strides)) and (shape[1] == 1 or strides[1] <= 1 << 22)


def _vec16(t):
    """t, or a copy of it, such that _strides_fit and its first value lies on a multiple of 16 bytes"""
    if t.data_ptr() % 16 == 0 and ((t.is_contiguous() and t.numel()) or _strides_fit(t.shape, t.stride(), t.element_size())):
        return t                                 # dense with a head size that the library takes: 16 bytes at a time
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """for a key: None says the same in less time where a tensor is dense"""
    return None if t.is_contiguous() else t.stride()


def _counts(c, B, dev, what):
    if c is None:
        return None
    c = _abi.to_dev(c, torch.int32, dev)
    if c.shape != (B,):
        raise ValueError(f"roi_attention: {what} must be ({B},), one count per image")
    return c


@functools.lru_cache(maxsize=1024)
def _attn_plan(q_shape, k_shape, q_stride, k_stride, v_stride, g_stride, masks, mask_stride, scale, dtype, backward):
    """the call's description for the library and its workspace's size: by shapes alone; a stride None: dense"""
    B, Nq, Hq, D = q_shape
    dense = [(shape[1] * shape[2] * D, shape[2] * D, D) for shape in (q_shape, k_shape)]
    strides = [(d if st is None else st)[:3] for st, d in ((q_stride, dense[0]), (k_stride, dense[1]), (v_stride, dense[1]), (g_stride, dense[0]))]
    s = _abi.AttnShape(B, Nq, k_shape[1], Hq, k_shape[2], D, *strides[0], *strides[1], *strides[2], *strides[3], masks, *mask_stride[:2],
                       max(D, 1) ** -0.5 if scale is None else scale, _abi.TYPES[dtype])
    return s, load().dg_roi_attn_workspace_bytes(s, backward)


def _attn_args(q, k, v, q_counts, k_counts, mask):
    """checks and lays out what the forward and the backward pass have in common"""
    dev = _abi.device_of(q, k, v)
    if not (q.device == dev and k.device == dev and v.device == dev):
        q, k, v = q.to(dev), k.to(dev), v.to(dev)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("roi_attention: q (B,Nq,Hq,D), k and v (B,Nk,Hk,D)")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("roi_attention: q, k and v must all be float32 or all be bfloat16")
    B, Nq, Nk = q.shape[0], q.shape[1], k.shape[1]
    qc, kc = _counts(q_counts, B, dev, "q_counts"), _counts(k_counts, B, dev, "k_counts")
    if mask is None:
        return dev, _vec16(q), _vec16(k), _vec16(v), qc, kc, None, 0, (0, 0)
    if not isinstance(mask, torch.Tensor) or mask.device != dev:
        mask = torch.as_tensor(mask, device=dev)
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError("roi_attention: mask must be bool (or uint8: not 0 = may be seen)")
    if mask.dim() == 2:
        mask = mask[None]
    if mask.dim() != 3 or mask.shape[0] not in (1, B) or tuple(mask.shape[1:]) != (Nq, Nk):
        raise ValueError("roi_attention: mask must be (Nq,Nk) or (B or 1,Nq,Nk)")
    if Nk > 1 and mask.stride(2) != 1:
        mask = mask.contiguous()
    return dev, _vec16(q), _vec16(k), _vec16(v), qc, kc, mask, mask.shape[0], mask.stride()


def roi_attention(q, k, v, q_counts=None, k_counts=None, mask=None, scale=None, rest=False):
    """Attention over padded sets of RoIs or map cells: q (B,Nq,Hq,D), k and v (B,Nk,Hk,D), float32 or bfloat16, any strides,
    Hq a multiple of Hk (query head h reads key head h // (Hq // Hk)), D a multiple of 8 up to 128 -> out (B,Nq,Hq,D),
    lse (B,Hq,Nq) float32.  A row sees the keys before k_counts (B) of its image for which mask (B or 1,Nq,Nk) is not 0; scale
    defaults to D ** -0.5.  Rows that see nothing, rows behind q_counts (B) among them: out 0, lse -inf.  rest: -> out,
    lse, rest, what rounding took from a bfloat16 out (None in float32), for roi_attention_backward.  No reference counterpart.
    For a gradient: fast_rcnn.roi_attention."""
    r = _attn_forward(_attn_args(q, k, v, q_counts, k_counts, mask), scale, rest)
    return r if rest else r[:2]


def _attn_forward(args, scale, keep_rest):
    dev, q, k, v, qc, kc, mask, masks, ms = args
    s, nbytes = _attn_plan(q.shape, k.shape, _strides(q), _strides(k), _strides(v), None, masks, ms, None if scale is None else float(scale), q.dtype, 0)
    out = _empty_like(q)
    lse = q.new_empty((s.batch, s.q_heads, s.nq), dtype=torch.float32)
    rest = _empty_like(q) if keep_rest and q.dtype == torch.bfloat16 else None
    ws = _scratch(nbytes, q)
    _call(dev, load().dg_roi_attn_fwd, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), _at(qc), _at(kc), _at(mask), out.data_ptr(), lse.data_ptr(), _at(rest),
          _at(ws), nbytes, _stream(dev))
    return out, lse, rest


def roi_attention_backward(grad_out, q, k, v, out, lse, q_counts=None, k_counts=None, mask=None, scale=None, need_q=True, need_kv=True, rest=None):
    """Gradients of roi_attention from its inputs, out and lse, with the probabilities recomputed: dq (B,Nq,Hq,D), dk and dv
    (B,Nk,Hk,D), rows behind a count 0.  need_q / need_kv False leaves those out (None).  rest: roi_attention's; without it dq and
    dk of a bfloat16 call are off by up to 2^-8 of grad_out . out where a row sees few keys."""
    args = _attn_args(q, k, v, q_counts, k_counts, mask)
    dev, q = args[0], args[1]
    if not (grad_out.device == dev and out.device == dev and lse.device == dev):
        grad_out, out, lse = grad_out.to(dev), out.to(dev), lse.to(dev)
    if rest is not None:
        if rest.shape != q.shape or rest.dtype != q.dtype or q.dtype != torch.bfloat16:
            raise ValueError("roi_attention_backward: rest must have q's shape and be bfloat16, as q")
        rest = _vec16(rest.to(dev).contiguous())
    if grad_out.shape != q.shape or out.shape != q.shape or grad_out.dtype != q.dtype or out.dtype != q.dtype:
        raise ValueError("roi_attention_backward: grad_out and out must have q's shape and type")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32:
        raise ValueError("roi_attention_backward: lse must be (B,Hq,Nq) float32")
    return _attn_backward(args, grad_out, _vec16(out.contiguous()), lse.contiguous(), rest, scale, need_q, need_kv)


def _attn_backward(args, g, out, lse, rest, scale, need_q, need_kv):
    dev, q, k, v, qc, kc, mask, masks, ms = args
    g = _vec16(g)
    s, nbytes = _attn_plan(q.shape, k.shape, _strides(q), _strides(k), _strides(v), _strides(g), masks, ms, None if scale is None else float(scale), q.dtype, 1)
    dq = _empty_like(q) if need_q else None
    dk, dv = (_empty_like(k), _empty_like(k)) if need_kv else (None, None)
    ws = _scratch(nbytes, q)
    _call(dev, load().dg_roi_attn_bwd, s, g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _at(rest), _at(qc), _at(kc),
          _at(mask), _at(dq), _at(dk), _at(dv), _at(ws), nbytes, _stream(dev))
    return dq, dk, dv


# ------------------------------------------------------------------ RoI head: rotary positions
class RopePlan:
    """Which axis turns each pair of a head and how fast: made once (rope_plan), kept by the program, used by every call."""

    def __init__(self, turns, axis, axes, pairing):
        self.turns, self.axis, self.axes, self.pairing = turns, axis, axes, pairing
        self.pairs = turns.shape[0]

    def to(self, device):
        return self if self.turns.device == device else RopePlan(self.turns.to(device), self.axis.to(device), self.axes, self.pairing)


def rope_plan(sections, theta=10000.0, ladder="axis", pairing="halves", device=None):
    """sections: pairs of a head that each axis turns, e.g. (16, 24, 24) for frame, row and column of a head of 128.
    ladder "axis": an axis's i-th of m pairs turns by theta ** (-i / m) radians per unit of its position; "shared": the j-th of
    all pairs by theta ** (-j / sum(sections)).  pairing "halves": values j and j + sum(sections) form pair j; "neighbours":
    values 2 j and 2 j + 1."""
    sections = [int(m) for m in sections]
    if not 1 <= len(sections) <= 16 or min(sections) < 0 or sum(sections) < 1:
        raise ValueError("rope_plan: 1 to 16 axes, each with 0 or more pairs, one at least in all")
    if ladder not in ("axis", "shared") or pairing not in ("halves", "neighbours"):
        raise ValueError("rope_plan: ladder is 'axis' or 'shared', pairing 'halves' or 'neighbours'")
    theta = float(theta)
    if not 0.0 < theta < float("inf"):
        raise ValueError("rope_plan: theta must be positive and finite")
    n = sum(sections)
    step = [i / m for m in sections for i in range(m)] if ladder == "axis" else [j / n for j in range(n)]
    turns = torch.tensor([theta ** -e / (2.0 * math.pi) for e in step], dtype=torch.float64)
    axis = torch.tensor([a for a, m in enumerate(sections) for _ in range(m)], dtype=torch.int32)
    dev = torch.device(device) if device is not None else _abi.require_gpu()
    return RopePlan(turns.to(dev), axis.to(dev), len(sections), pairing)


def _dense_last(t):
    return t if t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


@functools.lru_cache(maxsize=1024)
def _rope_shape(q_shape, k_heads, pairs, axes, q_stride, k_stride, pos_batch, pos_row, dtype, pos64, pairing):
    B, N, Hq, D = q_shape
    return _abi.RopeShape(B, N, Hq, k_heads, D, pairs, axes, *q_stride[:3], *k_stride[:3], pos_batch, pos_row, _abi.TYPES[dtype],
                          _abi.F64 if pos64 else _abi.F32, _abi.ROPE_HALVES if pairing == "halves" else _abi.ROPE_NEIGHBOURS)


def rope_axes(q, pos, plan, k=None, inverse=False):
    """Turns the pairs of q (B,N,H,D) (and of k (B,N,Hk,D) in the same launch) by the positions pos (B,N,A) or (N,A) of their
    tokens as plan says; inverse: back, which is the gradient.  float32, bfloat16 or float16; values behind the plan's pairs are
    copied; float32 or float64 positions are used as they are, whole numbers as float64.  -> the turned q, or (q, k).  No
    reference counterpart.  For a gradient: fast_rcnn.rope_axes."""
    q, k = _rope_turn(*_rope_args(q, k, pos, plan), inverse)
    return q if k is None else (q, k)


def _rope_args(q, k, pos, plan):
    dev = _abi.device_of(q, k, pos)
    q = q if q.device == dev else q.to(dev)
    k = k if k is None or k.device == dev else k.to(dev)
    if not isinstance(pos, torch.Tensor) or pos.device != dev:
        pos = torch.as_tensor(pos, device=dev)
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or k.dtype != q.dtype)):
        raise ValueError("rope_axes: q (B,N,Hq,D), k (B,N,Hk,D) of one type")
    if q.dtype not in _abi.TYPES:
        raise ValueError("rope_axes: float32, bfloat16 or float16")
    if pos.requires_grad:
        raise ValueError("rope_axes: positions have no gradient here; detach them")
    if not pos.is_floating_point():
        pos = pos.to(torch.float64)
    elif pos.dtype not in (torch.float32, torch.float64):
        pos = pos.to(torch.float32)
    B, N = q.shape[:2]
    plan = plan.to(dev)
    if pos.dim() not in (2, 3) or tuple(pos.shape[-2:]) != (N, plan.axes) or (pos.dim() == 3 and pos.shape[0] not in (1, B)):
        raise ValueError(f"rope_axes: pos must be (B,N,{plan.axes}) or (N,{plan.axes})")
    return dev, q, k, _dense_last(pos), plan


def _rope_turn(dev, q, k, pos, plan, inverse):
    q, k = _dense_last(q), None if k is None else _dense_last(k)
    s = _rope_shape(q.shape, 0 if k is None else k.shape[2], plan.pairs, plan.axes, q.stride(), (0, 0, 0) if k is None else k.stride(),
                    pos.stride(0) if pos.dim() == 3 and pos.shape[0] > 1 else 0, pos.stride(-2), q.dtype, pos.dtype == torch.float64, plan.pairing)
    out_q = _empty_like(q)
    out_k = None if k is None else _empty_like(k)
    _call(dev, load().dg_rope_axes, s, q.data_ptr(), _at(k), pos.data_ptr(), plan.turns.data_ptr(), plan.axis.data_ptr(), 1 if inverse else 0, out_q.data_ptr(),
          _at(out_k), _stream(dev))
    return out_q, out_k


# ------------------------------------------------------------------ RoI head: log probabilities of labels
def _logits(z, labels, what):
    dev = _abi.device_of(z, labels)
    if not isinstance(z, torch.Tensor) or z.device != dev:
        z = torch.as_tensor(z, device=dev)
    if z.dim() != 2 or z.shape[1] < 1 or z.dtype not in _abi.TYPES:
        raise ValueError(f"{what}: logits must be (n,C), C >= 1, float32, bfloat16 or float16")
    z = _dense_last(z)
    if labels is not None:
        labels = _abi.to_dev(labels, torch.int64, dev)
        if labels.shape != z.shape[:1]:
            raise ValueError(f"{what}: one label per row")
    return dev, z, labels


def class_logprobs(logits, labels=None, top=0):
    """logits (n,C) float32, bfloat16 or float16, labels (n) or None -> logp (n) of the labels (None without them), entropy (n),
    norm (n,2) (the row's maximum and the log of its sum of exponentials above it: what the gradient needs), top_logp (n,top),
    top_index (n,top) int64: the most probable classes, best first, equal logits by the lowest index (top 0 to 32).  A negative label gives none (logp 0, no gradient); a label of C or more gives NaN.  -inf is a masked class.
    No reference counterpart.  For a gradient: fast_rcnn.class_logprobs."""
    return _logprobs(*_logits(logits, labels, "class_logprobs"), int(top))


@functools.lru_cache(maxsize=1024)
def _logprobs_scratch(n, c, top):
    return load().dg_class_logprobs_workspace_bytes(n, c, top)


def _logprobs(dev, z, y, top):
    n, c = z.shape
    if not 0 <= top <= min(32, c):
        raise ValueError("class_logprobs: top must be 0 to 32 and no more than the classes")
    f32 = torch.float32
    entropy, norm = z.new_empty(n, dtype=f32), z.new_empty((n, 2), dtype=f32)
    logp = _empty_like(entropy) if y is not None else None
    best, index = z.new_empty((n, top), dtype=f32), z.new_empty((n, top), dtype=torch.int64)
    nbytes = _logprobs_scratch(n, c, top)
    ws = _scratch(nbytes, z)
    _call(dev, load().dg_class_logprobs, z.data_ptr(), _abi.TYPES[z.dtype], _at(y), n, c, z.stride(0), top, _at(logp), entropy.data_ptr(), norm.data_ptr(),
          best.data_ptr(), index.data_ptr(), None, _at(ws), nbytes, _stream(dev))
    return logp, entropy, norm, best, index


def class_logprobs_backward(grad_logp, grad_entropy, logits, labels, norm, entropy):
    """Gradient of the logits from those of logp and entropy (either may be None) and what class_logprobs gave."""
    dev, z, y = _logits(logits, labels, "class_logprobs_backward")
    n, c = z.shape
    args = []
    for t, shape in ((norm, (n, 2)), (entropy, (n,)), (grad_logp, (n,)), (grad_entropy, (n,))):
        t = None if t is None else _abi.to_dev(t, torch.float32, dev)
        if t is not None and t.shape != shape:
            raise ValueError("class_logprobs_backward: norm (n,2), entropy and the gradients (n)")
        args.append(t)
    return _logprobs_backward(dev, z, y, *args)


def _logprobs_backward(dev, z, y, norm, entropy, g, gh):
    n, c = z.shape
    dz = _empty_like(z)
    _call(dev, load().dg_class_logprobs_bwd, z.data_ptr(), _abi.TYPES[z.dtype], _at(y), n, c, z.stride(0), norm.data_ptr(), entropy.data_ptr(),
          _at(g) if y is not None else None, _at(gh), dz.data_ptr(), _stream(dev))
    return dz
