"""The sequence operators (``sam3_lora_amd.sequence``) as measured work: root-mean-square norm with the residual's addition and
an 8-bit output, rotary positions with several axes, and causal attention with grouped heads over packed sequences.

``run`` computes a case in plain torch operations in 32 bits where ``own`` is false, and calls the framework where it is true;
``exact`` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of a few requests: the norm in front of a frozen 8-bit projection, trunk width; latency
        dict(name="norm_q8_step", op="norm", rows=3, width=1024, type="bf16", residual=True, mode="q8", group=0),
        # a training step's norm over the tokens of eight images of 72 x 72 patches, gradients of the stream and the weight
        dict(name="norm_train", op="norm", rows=41472, width=1024, type="bf16", residual=True, mode="train", group=0),
        # a long prompt at a wide model, one scale for 128 values, an odd number of rows
        dict(name="norm_q8_prompt", op="norm", rows=16411, width=4096, type="bf16", residual=True, mode="q8", group=128),
        # one decoding step far into a sequence
        dict(name="rope_step", op="rope", tokens=7, heads=16, kv_heads=4, dim=64, type="bf16", mode="fwd", pairing="halves",
             spectrum="shared", axes="8,12,12", grid="far"),
        # eight frames of 72 x 72 patches, (time, height, width) each with a spectrum of its own, forward and backward
        dict(name="rope_video_train", op="rope", tokens=41472, heads=16, kv_heads=16, dim=64, type="bf16", mode="train",
             pairing="adjacent", spectrum="per_axis", axes="8,12,12", grid="video"),
        # fractional positions of an interpolated grid in 32 bits, a part of each head left unrotated, odd length
        dict(name="rope_f32_partial", op="rope", tokens=5183, heads=32, kv_heads=8, dim=128, type="f32", mode="fwd",
             pairing="halves", spectrum="shared", axes="24,24", grid="fraction"),
        # a batch of text prompts of 2 to 32 tokens through the text tower's attention, forward and backward
        dict(name="attn_text_train", op="attn", batch=96, q_low=2, q_high=32, extra=0, lens_seed=1, heads=16, kv_heads=16, dim=64,
             type="bf16", mode="train", causal=True),
        # one new token of each request over long caches of different lengths
        dict(name="attn_decode", op="attn", batch=24, q_low=1, q_high=1, extra=32767, lens_seed=2, heads=32, kv_heads=8, dim=128,
             type="bf16", mode="fwd", causal=True),
        # prompts of different lengths in one pack
        dict(name="attn_prefill", op="attn", batch=5, q_low=601, q_high=5184, extra=0, lens_seed=3, heads=32, kv_heads=8, dim=128,
             type="bf16", mode="fwd", causal=True),
        # queries that look at memories of other lengths, 32 bits, the detector's head size
        dict(name="attn_cross_f32_train", op="attn", batch=3, q_low=200, q_high=201, extra=901, lens_seed=4, heads=8, kv_heads=8,
             dim=32, type="f32", mode="train", causal=False),
        # the trunk's attention over whole images: every token sees every other
        dict(name="attn_grid_train", op="attn", batch=4, q_low=5184, q_high=5184, extra=0, lens_seed=5, heads=16, kv_heads=16,
             dim=64, type="bf16", mode="train", causal=False),
        # long packed documents with grouped heads, forward and backward
        dict(name="attn_long_train", op="attn", batch=2, q_low=6001, q_high=8192, extra=0, lens_seed=6, heads=32, kv_heads=8,
             dim=128, type="bf16", mode="train", causal=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "rope", "attn", "attn"])
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        width = 8 * _spread(rng, 8, 1024)
        rows = _spread(rng, 1, max(1, 67_000_000 // width))
        mode = rng.choice(["fwd", "train", "q8"])
        group = rng.choice([0, 32, 64, 128]) if mode == "q8" else 0
        return dict(op=op, rows=rows, width=width - width % group if group and width >= group else width, type=kind,
                    residual=rng.random() < 0.7, mode=mode, group=group if width >= max(group, 1) else 0)
    if op == "rope":
        dim = rng.choice([32, 64, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        n = rng.randint(1, 4)
        most = dim // 2
        axes = [max(1, int(most * rng.uniform(0.4, 1.0) / n)) for _ in range(n)]
        cap = 41472 * 32 * 64 // ((heads + kv) * dim * (2 if kind == "f32" else 1))
        return dict(op=op, tokens=_spread(rng, 1, min(41472, cap)), heads=heads, kv_heads=kv, dim=dim, type=kind,
                    mode=rng.choice(["fwd", "train"]), pairing=rng.choice(["adjacent", "halves"]),
                    spectrum=rng.choice(["shared", "per_axis"]), axes=",".join(str(a) for a in axes),
                    grid=rng.choice(["far", "video", "fraction"]))
    dim = rng.choice([32, 64, 64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7])
    causal = rng.random() < 0.7
    if rng.random() < 0.3:      # a decoding step
        batch = _spread(rng, 1, 24)
        extra = _spread(rng, 1, 20000)
        return dict(op=op, batch=batch, q_low=1, q_high=rng.choice([1, 1, 3]), extra=extra, lens_seed=rng.randrange(1 << 20),
                    heads=heads, kv_heads=kv, dim=dim, type=kind, mode="fwd", causal=True)
    batch = _spread(rng, 1, 48)
    longest = _spread(rng, 2, max(2, min(4096, int(4096 / math.sqrt(batch)))))
    if kind == "f32":
        longest = min(longest, 1500)
    return dict(op=op, batch=batch, q_low=_spread(rng, 1, longest), q_high=longest, extra=rng.choice([0, 0, 77]),
                lens_seed=rng.randrange(1 << 20), heads=heads, kv_heads=kv, dim=dim, type=kind,
                mode=rng.choice(["fwd", "train"]), causal=causal)


def _lengths(case):
    """(query lengths, key lengths) of the pack."""
    rng = random.Random(case["lens_seed"])
    lq = [rng.randint(case["q_low"], case["q_high"]) for _ in range(case["batch"])]
    return lq, [n + rng.randint(0, case["extra"]) for n in lq]


def _sections(case):
    return tuple(int(a) for a in case["axes"].split(","))


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "norm":
        n, c = case["rows"] * case["width"], case["width"]
        if case["mode"] == "q8":
            scales = case["rows"] * (c // case["group"] if case["group"] else 1)
            b = n * size + n + 4 * scales + (2 * n * size if case["residual"] else 0) + c * size
            return dict(bytes=b, flops=6 * n)
        fwd = (4 if case["residual"] else 2) * n * size + c * size
        if case["mode"] == "fwd":
            return dict(bytes=fwd, flops=5 * n)
        # backward: the gradients of y (and of the stream), the stream, one gradient out (both addends share it)
        return dict(bytes=fwd + (4 if case["residual"] else 3) * n * size + 2 * c * size, flops=16 * n)
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        pos = case["tokens"] * len(_sections(case)) * 4
        passes = 2 if case["mode"] == "train" else 1
        return dict(bytes=passes * (2 * n * size + pos), flops=passes * 3 * n)
    lq, lk = _lengths(case)
    if case["causal"]:
        pairs = sum(sum(max(0, min(k, i + k - q + 1)) for i in range(q)) for q, k in zip(lq, lk))
    else:
        pairs = sum(q * k for q, k in zip(lq, lk))
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    rows_q, rows_k = sum(lq) * h * d * size, sum(lk) * hk * d * size
    if case["mode"] == "fwd":
        return dict(bytes=2 * rows_q + 2 * rows_k, flops=4 * pairs * h * d)
    return dict(bytes=2 * rows_q + 2 * rows_k + 2 * rows_q + 2 * rows_k, flops=14 * pairs * h * d)


# ----------------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape, type, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(TYPES[type])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, train = case["type"], case["mode"] == "train"
    s = dict(case=case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        gain = torch.exp(0.5 * torch.randn(width, generator=g, device=DEVICE))     # a stream has loud and quiet channels
        s["x"] = (torch.randn(rows, width, generator=g, device=DEVICE) * gain).to(TYPES[kind])
        s["residual"] = (torch.randn(rows, width, generator=g, device=DEVICE) * 3 * gain).to(TYPES[kind]) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(width, generator=g, device=DEVICE)).to(TYPES[kind])
        if train:
            s["gy"] = _normal(g, rows, width, type=kind)
            s["gh"] = _normal(g, rows, width, type=kind) if case["residual"] else None
            for name in ("x", "residual", "weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif case["op"] == "rope":
        n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = _normal(g, n, h + 2 * hk, d, type=kind)          # the fused projection's output; q and k are views of it
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + hk]
        axes = len(_sections(case))
        t = torch.arange(n, device=DEVICE)
        if case["grid"] == "far":
            first = torch.randint(0, 1 << 20, (1, 1), generator=g, device=DEVICE)
            s["positions"] = (first + t).expand(axes, n).to(torch.int32).contiguous()
        else:
            grid = torch.stack([t // 5184, t % 5184 // 72, t % 72, t])[:axes]
            s["positions"] = grid.to(torch.int32) if case["grid"] == "video" else grid.float() * (24.0 / 72.0)
        if train:
            s["gq"], s["gk"] = _normal(g, n, h, d, type=kind), _normal(g, n, hk, d, type=kind)
            s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
    else:
        lq, lk = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s["q"] = _normal(g, sum(lq), h, d, type=kind, scale=1.5)
        s["k"], s["v"] = _normal(g, sum(lk), hk, d, type=kind), _normal(g, sum(lk), hk, d, type=kind)
        s["cu_q"], s["cu_k"] = _ends(lq), _ends(lk)
        s["max_q"], s["max_k"] = max(lq), max(lk)
        if train:
            s["go"] = _normal(g, sum(lq), h, d, type=kind)
            for name in ("q", "k", "v"):
                s[name].requires_grad_(True)
    return s


def _ends(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(DEVICE)


# ------------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if case["op"] == "norm":
        return _norm_own(s) if own else _norm_plain(s)
    if case["op"] == "rope":
        return _rope_own(s) if own else _rope_plain(s)
    return _attn_own(s) if own else _attn_plain(s)


def _norm_own(s):
    from sam3_lora_amd import sequence
    case, x, r, w = s["case"], s["x"], s["residual"], s["weight"]
    if case["mode"] == "q8":
        return sequence.rms_norm_q8(x, w, residual=r, eps=EPS, group=case["group"])
    got = sequence.rms_norm(x, w, residual=r, eps=EPS)
    if case["mode"] == "fwd":
        return got
    if r is None:
        return (got,) + torch.autograd.grad(got, (x, w), s["gy"])
    return got + torch.autograd.grad(got, (x, r, w), (s["gy"], s["gh"]))


def _norm_plain(s):
    case, kind = s["case"], TYPES[s["case"]["type"]]
    with torch.no_grad():
        w = s["weight"].float()
        h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        xhat = h * rstd
        y = xhat * w
        stream = () if s["residual"] is None else (h.to(kind),)
        if case["mode"] == "q8":
            parts = y.unflatten(-1, (-1, case["group"] or case["width"]))
            scale = parts.abs().amax(-1).clamp_min(2.0 ** -24) / E4M3_MAX
            image = (parts / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).flatten(-2).to(torch.float8_e4m3fn)
            return (image, scale) + stream
        out = (y.to(kind),) + stream
        if case["mode"] == "fwd":
            return out if stream else out[0]
        gy = s["gy"].float()
        gxhat = gy * w
        gh = rstd * (gxhat - xhat * (gxhat * xhat).mean(-1, keepdim=True))
        gw = (gy * xhat).sum(0).to(kind)
        if not stream:
            return out + (gh.to(kind), gw)
        gx = (gh + s["gh"].float()).to(kind)
        return out + (gx, gx, gw)


def _rope_own(s):
    from sam3_lora_amd import sequence
    case = s["case"]
    got = sequence.rotary_axes(s["q"], s["k"], s["positions"], _sections(case), theta=10000.0, pairing=case["pairing"],
                               spectrum=case["spectrum"])
    if case["mode"] == "fwd":
        return got
    return got + torch.autograd.grad(got, (s["q"], s["k"]), (s["gq"], s["gk"]))


def _rates(case):
    """(axis, angle for one step) of each rotated pair, as lists."""
    sections, dim = _sections(case), case["dim"]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if case["spectrum"] == "shared":
        return axis, [10000.0 ** (-i / sum(sections)) for i in range(len(axis))]
    return axis, [10000.0 ** (-i / n) for n in sections for i in range(n)]


def _turned(x, cos, sin, pairing):
    rot, rest = x[..., :2 * cos.shape[-1]].float(), x[..., 2 * cos.shape[-1]:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if pairing == "adjacent" else rot.chunk(2, -1)
    c, d = a * cos - b * sin, a * sin + b * cos
    both = torch.stack((c, d), -1).flatten(-2) if pairing == "adjacent" else torch.cat((c, d), -1)
    return torch.cat((both.to(x.dtype), rest), -1)


def _rope_plain(s):
    case = s["case"]
    with torch.no_grad():
        axis, rate = _rates(case)
        angle = s["positions"].double()[axis].t() * torch.tensor(rate, dtype=torch.float64, device=DEVICE)
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        out = _turned(s["q"], cos, sin, case["pairing"]), _turned(s["k"], cos, sin, case["pairing"])
        if case["mode"] == "fwd":
            return out
        return out + (_turned(s["gq"], cos, -sin, case["pairing"]), _turned(s["gk"], cos, -sin, case["pairing"]))


def _attn_own(s):
    from sam3_lora_amd import sequence
    out = sequence.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q=s["max_q"], max_k=s["max_k"],
                                    causal=s["case"]["causal"])
    if s["case"]["mode"] == "fwd":
        return out
    return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["go"])


def _padded(x, cu, longest):
    """[total, heads, dim] -> 32-bit [batch, heads, longest, dim], zeros behind each sequence."""
    at = torch.arange(longest, device=DEVICE)
    row = cu[:-1, None] + at
    inside = row < cu[1:, None]
    return (x[row.clamp(max=x.shape[0] - 1)].float() * inside[..., None, None]).transpose(1, 2).contiguous()


def _packed(x, cu, total, kind):
    """The inverse of `_padded`."""
    t = torch.arange(total, device=DEVICE)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True, out_int32=True)
    return x[seq, :, t - cu[seq]].to(kind)


def _attn_plain(s):
    case, kind = s["case"], TYPES[s["case"]["type"]]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    with torch.no_grad():
        cu_q, cu_k, nq, nk = s["cu_q"], s["cu_k"], s["max_q"], s["max_k"]
        grouped = lambda t: _padded(t, cu_q, nq).unflatten(1, (hk, h // hk)).flatten(2, 3)      # noqa: E731
        q, k, v = grouped(s["q"]), _padded(s["k"], cu_k, nk), _padded(s["v"], cu_k, nk)
        p = q @ k.transpose(-1, -2)
        p *= 1 / math.sqrt(d)
        lq, lk = (cu_q[1:] - cu_q[:-1])[:, None, None], (cu_k[1:] - cu_k[:-1])[:, None, None]
        i, j = torch.arange(nq, device=DEVICE)[:, None], torch.arange(nk, device=DEVICE)
        hidden = (j >= lk) | (i >= lq)
        if case["causal"]:
            hidden = hidden | (j > i + lk - lq)
        p.unflatten(2, (h // hk, nq)).masked_fill_(hidden[:, None, None], float("-inf"))
        p -= p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
        p.exp_()
        p /= p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
        back = lambda t: _packed(t.unflatten(2, (h // hk, nq)).flatten(1, 2), cu_q, s["q"].shape[0], kind)      # noqa: E731
        o = p @ v
        if case["mode"] == "fwd":
            return back(o)
        go = grouped(s["go"])
        gv = p.transpose(-1, -2) @ go
        ds = go @ v.transpose(-1, -2)
        ds -= (go * o).sum(-1, keepdim=True)
        ds *= p
        ds *= 1 / math.sqrt(d)
        gq, gk = ds @ k, ds.transpose(-1, -2) @ q
        return back(o), back(gq), _packed(gk, cu_k, s["k"].shape[0], kind), _packed(gv, cu_k, s["v"].shape[0], kind)


# --------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return dict(norm=_norm_exact, rope=_rope_exact, attn=_attn_exact)[case["op"]](case, s)


def _norm_exact(case, s):
    x, w, r = s["x"].double(), s["weight"].double(), s["residual"]
    h = x if r is None else x + r.double()
    length = (h.pow(2).sum(1) / case["width"] + EPS).sqrt()
    y = h / length[:, None] * w
    tail = [] if r is None else [h]
    if case["mode"] == "q8":
        g = case["group"] or case["width"]
        scale = (y.abs().reshape(case["rows"], -1, g).max(2).values / E4M3_MAX).clamp(min=2.0 ** -24 / E4M3_MAX)
        return [y / scale.repeat_interleave(g, 1), scale] + tail
    if case["mode"] == "fwd":
        return [y] + tail if tail else y
    gy = s["gy"].double()
    u = gy * w
    along = (u * h).sum(1) / case["width"]
    gh = u / length[:, None] - h * (along / length.pow(3))[:, None]
    if tail:
        gh = gh + s["gh"].double()
    gw = (gy * h / length[:, None]).sum(0)
    return [y] + tail + ([gh, gh, gw] if tail else [gh, gw])


def _rope_exact(case, s):
    sections = _sections(case)
    n = sum(sections)
    rate, start = [], 0
    for a, m in enumerate(sections):
        for i in range(m):
            rate.append((a, 10000.0 ** (-(start + i) / n if case["spectrum"] == "shared" else -i / m)))
        start += m
    first = [2 * i if case["pairing"] == "adjacent" else i for i in range(n)]
    second = [2 * i + 1 if case["pairing"] == "adjacent" else i + n for i in range(n)]
    pos = s["positions"].double()
    turn = torch.polar(torch.ones(case["tokens"], n, dtype=torch.float64, device=DEVICE),
                       torch.stack([pos[a] * f for a, f in rate], 1))[:, None]

    def apply(x, turn):
        x = x.detach().double().clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = [apply(s["q"], turn), apply(s["k"], turn)]
    if case["mode"] == "train":
        out += [apply(s["gq"], turn.conj()), apply(s["gk"], turn.conj())]
    return out


def _attn_exact(case, s):
    lq, lk = _lengths(case)
    group, c = case["heads"] // case["kv_heads"], 1 / math.sqrt(case["dim"])
    train = case["mode"] == "train"
    names = ["q", "q", "k", "v"] if train else ["q"]
    outs = [torch.zeros(s[n].shape, dtype=torch.float64, device=DEVICE) for n in names]
    a = b = 0
    for m, n in zip(lq, lk):
        seen = torch.ones(m, n, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            seen = seen.tril(n - m)
        for head in range(case["heads"]):
            kv = head // group
            q, k, v = s["q"][a:a + m, head].double(), s["k"][b:b + n, kv].double(), s["v"][b:b + n, kv].double()
            p = torch.softmax((q @ k.T * c).masked_fill(~seen, -math.inf), 1).nan_to_num(0.0)
            o = p @ v
            outs[0][a:a + m, head] = o
            if train:
                go = s["go"][a:a + m, head].double()
                ds = p * (go @ v.T - (go * o).sum(1, keepdim=True)) * c
                outs[1][a:a + m, head] = ds @ k
                outs[2][b:b + n, kv] += ds.T @ q
                outs[3][b:b + n, kv] += p.T @ go
        a, b = a + m, b + n
    return outs if train else outs[0]
