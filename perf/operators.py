"""Measured cases of the RoI head's operators: rotary positions over several axes, attention over padded sets of RoIs or map
cells (forward, and a training step with its backward pass), and log probabilities of labels with entropy and top classes.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) where `own` is
false, and calls the framework's operator where it is true."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # attention, forward only ("infer") and with its backward pass ("train")
        # the 98 boxes of one YOLOv1 image related to each other: the smallest call, where latency counts
        dict(name="attn infer 98 boxes", op="attn", train=False, dtype="bf16", b=1, nq=98, nk=98, hq=4, hk=4, d=32, ragged=False, mask="none"),
        # 16 images of up to 2000 proposals each, as many as every image has
        dict(name="attn infer 16x2000 rois", op="attn", train=False, dtype="bf16", b=16, nq=2000, nk=2000, hq=8, hk=8, d=64, ragged=True, mask="none"),
        # one tracked object per stream looks its past up in a long memory of box features, heads shared by four
        dict(name="attn infer 1 over 120001", op="attn", train=False, dtype="bf16", b=2, nq=1, nk=120001, hq=8, hk=2, d=128, ragged=True, mask="none"),
        # proposals against the 38x50 cells of the feature map, training
        dict(name="attn train 2000 to 1900", op="attn", train=True, dtype="bf16", b=8, nq=2000, nk=1900, hq=8, hk=8, d=64, ragged=True, mask="none"),
        # proposals that may only see those they overlap (some see none), single precision as the pooled features come
        dict(name="attn train 509 masked fp32", op="attn", train=True, dtype="fp32", b=4, nq=509, nk=509, hq=8, hk=2, d=64, ragged=True, mask="pairs"),
        # the boxes of a whole clip at once: the largest
        dict(name="attn train 16001", op="attn", train=True, dtype="bf16", b=1, nq=16001, nk=16001, hq=8, hk=8, d=128, ragged=False, mask="none"),
        # rotary positions: row and column of 98 boxes, one image
        dict(name="rope infer 98 boxes", op="rope", train=False, dtype="bf16", b=1, n=98, hq=4, hk=4, d=32, axes=2, far=False, pairing="halves"),
        # row and column of 16 images' proposals, single precision, part of each head left unturned
        dict(name="rope train 16x2000 fp32", op="rope", train=True, dtype="fp32", b=16, n=2000, hq=8, hk=8, d=80, axes=2, far=False, pairing="neighbours"),
        # frame, row and column of 16 frames of 38x50 cells in four clips
        dict(name="rope train 4x30400 cells", op="rope", train=True, dtype="bf16", b=4, n=30400, hq=16, hk=4, d=128, axes=3, far=True, pairing="halves"),
        # log probabilities: one object over a large open list of names, with the best eight
        dict(name="logp infer 1x131072", op="logp", train=False, dtype="bf16", n=1, c=131072, top=8),
        # the proposals of 16 images over 80 classes and background, with the gradient
        dict(name="logp train 32000x81", op="logp", train=True, dtype="fp32", n=32000, c=81, top=3),
        # a large hierarchy of classes, ragged length, with the gradient
        dict(name="logp train 8192x20011", op="logp", train=True, dtype="bf16", n=8192, c=20011, top=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rope", "logp"])
    if op == "attn":
        train = rng.random() < 0.6
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 1, 2, 4])
        d = rng.choice([32, 40, 64, 64, 80, 128])
        nq = 1 if rng.random() < 0.2 and not train else _log(rng, 2, 8000)
        nk = _log(rng, 16, 60000) if nq == 1 else nq if rng.random() < 0.5 else _log(rng, 2, 8000)
        b = _log(rng, 1, 32)
        while b > 1 and b * nq * nk * hq * d > 16001 * 16001 * 8 * 32:
            b -= 1
        return dict(op="attn", train=train, dtype=dtype, b=b, nq=nq, nk=nk, hq=hq, hk=hk, d=d, ragged=rng.random() < 0.5,
                    mask="pairs" if nq > 1 and b * nq * nk < 1 << 26 and rng.random() < 0.4 else "none")
    if op == "rope":
        n, b = _log(rng, 1, 30000), _log(rng, 1, 16)
        while b > 1 and b * n > 60000:
            b -= 1
        return dict(op="rope", train=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "fp32"]), b=b, n=n, hq=rng.choice([3, 4, 8, 16]),
                    hk=rng.choice([1, 2, 4]), d=rng.choice([32, 64, 80, 128]), axes=rng.choice([1, 2, 3]), far=rng.random() < 0.5,
                    pairing=rng.choice(["halves", "neighbours"]))
    c = _log(rng, 2, 131072)
    n = _log(rng, 1, max(1, min(65536, (1 << 27) // c)))
    return dict(op="logp", train=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "fp32"]), n=n, c=c, top=rng.randint(1, min(c, 8)))


def work(case):
    c, e = case, 4 if case["dtype"] == "fp32" else 2
    if c["op"] == "attn":
        q, kv = c["b"] * c["nq"] * c["hq"] * c["d"], c["b"] * c["nk"] * c["hk"] * c["d"]
        live = 0.75 if c["ragged"] else 1.0  # counts lie between a half and all of the rows, on both sides where both have several
        pairs = c["b"] * c["hq"] * (c["nq"] * (live if c["nq"] > 1 else 1.0)) * (c["nk"] * live)
        byt = (2 * q + 2 * kv * live) * e + c["b"] * c["hq"] * c["nq"] * 4
        if c["mask"] != "none":
            byt += c["b"] * c["nq"] * c["nk"]
        if c["train"]:
            byt += (2 * q + 2 * kv) * e
        return {"bytes": byt, "flops": pairs * c["d"] * (14 if c["train"] else 4)}
    if c["op"] == "rope":
        x = c["b"] * c["n"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": (4 if c["train"] else 2) * x * e + c["b"] * c["n"] * c["axes"] * 4, "flops": (6 if c["train"] else 3) * x}
    z = c["n"] * c["c"]
    return {"bytes": (2 if c["train"] else 1) * z * e + c["n"] * (8 + 8 + 12 * c["top"] + (8 if c["train"] else 0)), "flops": (10 if c["train"] else 6) * z}


# ------------------------------------------------------------------ inputs
def _sections(case):
    pairs = case["d"] // 2 if case["d"] != 80 else 32  # heads of 80 turn their first 64 values
    a = case["axes"]
    first = pairs // 4 if a == 3 else pairs // a
    rest = pairs - first
    return [pairs] if a == 1 else [first, rest] if a == 2 else [first, rest // 2, rest - rest // 2]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    s = {"case": case}
    if case["op"] == "attn":
        b, nq, nk, hq, hk, d = (case[k] for k in ("b", "nq", "nk", "hq", "hk", "d"))
        s["q"], s["k"], s["v"] = normal(b, nq, hq, d), normal(b, nk, hk, d), normal(b, nk, hk, d)
        s["q_counts"] = s["k_counts"] = s["mask"] = None
        if case["ragged"]:
            s["k_counts"] = torch.randint(nk - nk // 2, nk + 1, (b,), generator=g, device=dev, dtype=torch.int32)
            if nq > 1:
                s["q_counts"] = s["k_counts"] if nq == nk else torch.randint(nq - nq // 2, nq + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        if case["mask"] == "pairs":  # a row sees about a fifth of the others, and one row in 32 nobody
            m = torch.rand((b, nq, nk), generator=g, device=dev) < 0.2
            s["mask"] = m & (torch.rand((b, nq, 1), generator=g, device=dev) > 1 / 32)
        if case["train"]:
            s["do"] = normal(b, nq, hq, d)
            for t in ("q", "k", "v"):
                s[t].requires_grad_(True)
    elif case["op"] == "rope":
        b, n, d = case["b"], case["n"], case["d"]
        s["q"], s["k"] = normal(b, n, case["hq"], d), normal(b, n, case["hk"], d)
        # centres in cells of a map of 38 x 50; the first of three axes is the frame's number, far into a recording where `far`
        pos = torch.rand((b, n, case["axes"]), generator=g, device=dev) * torch.tensor([38.0, 50.0, 50.0][:case["axes"]], device=dev)
        if case["axes"] == 3 or case["far"]:
            start = torch.randint(0, 200000 if case["far"] else 64, (b, 1), generator=g, device=dev)
            pos[:, :, 0] = (start + torch.arange(n, device=dev)[None, :] // 1900).float()
        s["pos"] = pos
        if case["train"]:
            s["dq"], s["dk"] = normal(b, n, case["hq"], d), normal(b, n, case["hk"], d)
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        if own:
            from vision_amd import ops
            s["plan"] = ops.rope_plan(_sections(case), theta=10000.0, pairing=case["pairing"], device=dev)
        else:
            s["freq"], s["axis"] = _ladder(case, dev)
    else:
        n, c = case["n"], case["c"]
        z = torch.randn((n, c), generator=g, device=dev, dtype=torch.float32) * 2.0
        z += 4.0 * torch.randn((1, c), generator=g, device=dev, dtype=torch.float32).clamp(max=1.0)  # some classes are rare
        s["z"] = z.to(dt)
        s["y"] = torch.randint(0, c, (n,), generator=g, device=dev)
        s["y"][torch.rand((n,), generator=g, device=dev) < 0.02] = -1  # padded rows carry no label
        if case["train"]:
            s["g"] = torch.rand((n,), generator=g, device=dev) / n * -1.0
            s["gh"] = torch.randn((n,), generator=g, device=dev) * (0.01 / n)
            s["z"].requires_grad_(True)
    return s


def _ladder(case, dev):
    """radians per unit of position and the axis of each pair: an axis's i-th of m pairs turns by 10000^(-i/m)"""
    sec = _sections(case)
    freq = torch.cat([10000.0 ** (-torch.arange(m, dtype=torch.float64, device=dev) / m) for m in sec])
    return freq, torch.cat([torch.full((m,), a, dtype=torch.int64, device=dev) for a, m in enumerate(sec)])


# ------------------------------------------------------------------ one pass
def run(state):
    return {"attn": _attn, "rope": _rope, "logp": _logp}[state["case"]["op"]](state)


def _attn(s):
    train = s["case"]["train"]
    if own:
        from vision_amd import fast_rcnn, ops
        more = dict(q_counts=s["q_counts"], k_counts=s["k_counts"], mask=s["mask"])
        if not train:
            out, lse = ops.roi_attention(s["q"], s["k"], s["v"], **more)
            return {"out": out, "lse": lse}
        out = fast_rcnn.roi_attention(s["q"], s["k"], s["v"], **more)
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return _attn_plain(s, train)


def _seen(s, nq, nk, dev):
    """(b or 1, 1, 1, nq, nk) truth values: which key each row may see; None: all"""
    see = None
    if s["k_counts"] is not None:
        see = (torch.arange(nk, device=dev)[None, :] < s["k_counts"][:, None])[:, None, :]
    if s["q_counts"] is not None:
        live = (torch.arange(nq, device=dev)[None, :] < s["q_counts"][:, None])[:, :, None]
        see = live if see is None else see & live
    if s["mask"] is not None:
        see = s["mask"] if see is None else see & s["mask"]
    return None if see is None else see[:, None, None]


def _attn_plain(s, train):
    q, k, v = s["q"], s["k"], s["v"]
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d)
    qf = q.float().view(b, nq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).contiguous()
    kf, vf = (t.float().permute(0, 2, 1, 3)[:, :, None].contiguous() for t in (k, v))
    see = _seen(s, nq, nk, q.device)
    x = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale)
    if see is not None:
        x.masked_fill_(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = top + total.log()
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = torch.matmul(p, vf)

    def rows(t, n):
        return t.permute(0, 3, 1, 2, 4).reshape(b, n, -1, d).to(q.dtype)

    if not train:
        return {"out": rows(out, nq), "lse": lse.reshape(b, hq, nq)}
    do = s["do"].float().view(b, nq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).contiguous()
    if s["q_counts"] is not None:
        do = do * (torch.arange(nq, device=q.device)[None, :] < s["q_counts"][:, None])[:, None, None, :, None]
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    dp = torch.matmul(do, vf.transpose(-1, -2))
    delta = (p * dp).sum(-1, keepdim=True)
    ds = dp.sub_(delta).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kf)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2, keepdim=True)
    return {"out": rows(out, nq), "dq": rows(dq, nq), "dk": rows(dk, nk), "dv": rows(dv, nk)}


def _rope(s):
    train = s["case"]["train"]
    if own:
        from vision_amd import fast_rcnn, ops
        if not train:
            q, k = ops.rope_axes(s["q"], s["pos"], s["plan"], k=s["k"])
            return {"q": q, "k": k}
        q, k = fast_rcnn.rope_axes(s["q"], s["k"], s["pos"], s["plan"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    with torch.no_grad():
        angle = s["pos"].double()[:, :, s["axis"]] * s["freq"]
        cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
        pairing = s["case"]["pairing"]
        out = {"q": _turn(s["q"], cos, sin, pairing), "k": _turn(s["k"], cos, sin, pairing)}
        if train:
            out.update(dq=_turn(s["dq"], cos, -sin, pairing), dk=_turn(s["dk"], cos, -sin, pairing))
        return out


def _turn(x, cos, sin, pairing):
    r, y = cos.shape[-1], x.float()
    u, v = (y[..., :r], y[..., r:2 * r]) if pairing == "halves" else (y[..., 0:2 * r:2], y[..., 1:2 * r:2])
    a, b = u * cos - v * sin, u * sin + v * cos
    turned = torch.cat([a, b], -1) if pairing == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, y[..., 2 * r:]], -1).to(x.dtype)


def _logp(s):
    top, train = s["case"]["top"], s["case"]["train"]
    if own:
        from vision_amd import fast_rcnn, ops
        if not train:
            logp, entropy, _, best, index = ops.class_logprobs(s["z"], s["y"], top=top)
            return {"logp": logp, "entropy": entropy, "best": best, "index": index}
        r = fast_rcnn.class_logprobs(s["z"], s["y"], top=top)
        (dz,) = torch.autograd.grad((r.logp, r.entropy), (s["z"],), (s["g"], s["gh"]))
        return {"logp": r.logp, "entropy": r.entropy, "best": r.top_logp, "index": r.top_index, "dz": dz}
    with torch.no_grad():
        return _logp_plain(s, top, train)


def _logp_plain(s, top, train):
    z, y = s["z"].float(), s["y"]
    n, c = z.shape
    peak = z.amax(1, keepdim=True)
    e = (z - peak).exp()
    total = e.sum(1, keepdim=True)
    lse = peak + total.log()
    lp = z - lse
    p = e / total
    entropy = -(p * lp).sum(1)
    known = y >= 0
    logp = torch.where(known, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros_like(entropy))
    bits = (lp + 0.0).view(torch.int32).long()  # ordered as the values are; equal ones by the lowest index
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + (c - 1 - torch.arange(c, device=z.device))
    index = torch.topk(key, top, dim=1).indices
    out = {"logp": logp, "entropy": entropy, "best": lp.gather(1, index), "index": index}
    if train:
        g = torch.where(known, s["g"], torch.zeros_like(s["g"]))
        dz = -p * (g[:, None] + s["gh"][:, None] * (lp + entropy[:, None]))
        dz.scatter_add_(1, y.clamp(min=0)[:, None], g[:, None])
        out["dz"] = dz.to(s["z"].dtype)
    return out


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "rope": _exact_rope, "logp": _exact_logp}[case["op"]](case, s)


def _exact_attn(case, s):
    b, nq, nk, hq, hk, d = (case[x] for x in ("b", "nq", "nk", "hq", "hk", "d"))
    dev = s["q"].device
    f64 = dict(dtype=torch.float64, device=dev)
    out, lse = torch.zeros(b, nq, hq, d, **f64), torch.full((b, hq, nq), -math.inf, **f64)
    dq, dk, dv = torch.zeros(b, nq, hq, d, **f64), torch.zeros(b, nk, hk, d, **f64), torch.zeros(b, nk, hk, d, **f64)
    for i in range(b):
        rows = nq if s["q_counts"] is None else int(s["q_counts"][i])
        keys = nk if s["k_counts"] is None else int(s["k_counts"][i])
        for h in range(hq):
            kv = h // (hq // hk)
            q, k, v = s["q"][i, :rows, h].double(), s["k"][i, :keys, kv].double(), s["v"][i, :keys, kv].double()
            x = (q @ k.T) * d ** -0.5
            if s["mask"] is not None:
                x[~s["mask"][i, :rows, :keys]] = -math.inf
            full = torch.logsumexp(x, 1)
            lse[i, h, :rows] = full
            p = torch.exp(x - torch.where(torch.isinf(full), 0.0, full)[:, None])
            o = p @ v
            out[i, :rows, h] = o
            if case["train"]:
                do = s["do"][i, :rows, h].double()
                dv[i, :keys, kv] += p.T @ do
                t = p * (do @ v.T - (do * o).sum(1, keepdim=True)) * d ** -0.5
                dq[i, :rows, h] = t @ k
                dk[i, :keys, kv] += t.T @ q
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"out": out, "lse": lse}


def _exact_rope(case, s):
    sec, pos = _sections(case), s["pos"].double()
    pairs = sum(sec)

    def complex_turn(x, sign):
        z = x.double()
        head = z[..., :2 * pairs]
        w = torch.complex(head[..., :pairs], head[..., pairs:]) if case["pairing"] == "halves" else torch.complex(head[..., ::2], head[..., 1::2])
        parts, at = [], 0
        for a, m in enumerate(sec):
            f = torch.exp(torch.arange(m, dtype=torch.float64, device=z.device) * (-math.log(10000.0) / m))
            turn = sign * pos[:, :, None, a:a + 1] * f
            parts.append(w[..., at:at + m] * torch.polar(torch.ones_like(turn), turn))
            at += m
        w = torch.cat(parts, -1)
        y = z.clone()
        if case["pairing"] == "halves":
            y[..., :pairs], y[..., pairs:2 * pairs] = w.real, w.imag
        else:
            y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = w.real, w.imag
        return y

    out = {"q": complex_turn(s["q"], 1.0), "k": complex_turn(s["k"], 1.0)}
    if case["train"]:
        out.update(dq=complex_turn(s["dq"], -1.0), dk=complex_turn(s["dk"], -1.0))
    return out


def _exact_logp(case, s):
    z, y, t = s["z"].double(), s["y"], case["top"]
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    entropy = -(p * lp).sum(1)
    row = torch.arange(case["n"], device=z.device)
    known = y >= 0
    logp = torch.zeros_like(entropy)
    logp[known] = lp[row[known], y[known]]
    out = {"logp": logp, "entropy": entropy, "best": torch.topk(lp, t, dim=1).values, "index": None}
    if case["train"]:
        hot = torch.zeros_like(p)
        hot[row[known], y[known]] = 1.0
        g = torch.where(known, s["g"], 0.0).double()[:, None]
        out["dz"] = g * (hot - p) - s["gh"].double()[:, None] * p * (lp + entropy[:, None])
    return out
