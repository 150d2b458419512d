"""
Sequence operators (sam3_lora_amd/sequence.py, include/sam3_seq_amd.h) against their definitions in 64 bits.

Tolerances are sums of the roundings that a result passes through.  u = finfo(type).eps / 2 is the relative error of one rounding to
the activations' type (bf16 2^-8, fp32 2^-24), F = 2^-24 of one fp32 operation; a sum of n products in fp32 is off by at most
(n + 1) F times the sum of the products' absolute values, whatever its order.
"""
import math

import pytest
import torch

from sam3_lora_amd import _ffi, sequence
from sam3_lora_amd._ffi import LoRAKernelError

F = 2.0 ** -24
DT = [torch.bfloat16, torch.float32]
ids = lambda t: str(t).replace("torch.", "")      # noqa: E731


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, dtype, scale=1.0):
    """Values that the type holds exactly, on the CPU in 64 bits."""
    return (torch.randn(*shape, generator=g) * scale).to(dtype).double()


def close(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - tol
    assert (over <= 0).all(), f"{what}: off by {(got - want).abs().max().item():.3e}, {int((over > 0).sum())} beyond the bound, worst by {over.max().item():.3e}"


# ----------------------------------------------------------------------------------------------------------- refusals
def test_header_exports_and_error_text():
    import ctypes
    import os
    import re
    from sam3_lora_amd import build
    hdr = open(os.path.join(build.INCLUDE, "sam3_seq_amd.h")).read()
    assert set(re.findall(r"\b(sam3_seq_[a-z_0-9]+)\s*\(", hdr)) == set(_ffi.SEQ_EXPORTS)
    lib = _ffi.load()
    assert lib.sam3_seq_rms_norm_bwd_workspace_bytes(0, 64) == 0 == lib.sam3_seq_rms_norm_bwd_workspace_bytes(8, 63)
    assert lib.sam3_seq_rms_norm_bwd_workspace_bytes(3, 1024) == 1024 * 4
    assert lib.sam3_seq_attn_bwd_workspace_bytes(5, 4) == 240
    p = ctypes.c_void_p(64)

    def norm(M=1, C=64, dtype=0, x=p, w=p, y=p, q8=None, scales=None, group=0, fmt=0, eps=1e-6, ldx=64, low=None):
        return lib.sam3_seq_rms_norm_fwd(x, ldx, None, 0, w, y, None, low, None, q8, scales, group, fmt, M, C, eps, dtype, None)
    for bad, text in ((dict(dtype=2), "dtype"), (dict(C=60), "multiples of 8"), (dict(M=-1), "sizes"), (dict(x=None), "null"), (dict(y=None), "null"),
                      (dict(q8=p), "scales"), (dict(q8=p, scales=p, group=48), "groups"), (dict(q8=p, scales=p, fmt=3), "format"),
                      (dict(eps=-1.0), "eps"), (dict(ldx=32), "pitch"), (dict(low=p), "h_low"), (dict(x=ctypes.c_void_p(68)), "aligned")):
        assert norm(**bad) == -22, bad
        assert text in lib.sam3_seq_last_error().decode(), (bad, lib.sam3_seq_last_error())
    assert norm(C=16392, ldx=16392) == -95 and norm(M=0) == 0

    turns, axis = (ctypes.c_double * 16)(), (ctypes.c_ubyte * 16)()

    def rope(q=p, T=1, Hq=1, D=32, pairs=16, pos_type=0, axes=1, st=32, dtype=0):
        return lib.sam3_seq_rotary(q, st, 32, None, 0, 0, p, None, p, 0, 1, pos_type, axes, turns, axis, pairs, 0, 0, T, Hq, 0, D, dtype, None)
    for bad in (dict(q=None), dict(D=36), dict(pairs=17), dict(pairs=0), dict(pos_type=3), dict(axes=0), dict(st=33), dict(dtype=5), dict(Hq=0)):
        assert rope(**bad) == -22, bad
    assert rope(T=0) == 0 and rope(Hq=2000) == -95
    axis[3] = 1
    assert rope() == -22 and "axis" in lib.sam3_seq_last_error().decode()

    def attn(q=p, B=1, Hq=4, Hk=2, D=64, Tq=8, Tk=8, scale=0.1, dtype=0, st=64, cu=p):
        return lib.sam3_seq_attn_fwd(q, st, 64, p, 64, 64, p, 64, 64, cu, p, None, p, None, None, Tq, Tk, B, Hq, Hk, D, 8, 8, 1, scale, dtype, None, 0, None)
    for bad in (dict(q=None), dict(Hk=3), dict(D=60), dict(scale=0.0), dict(scale=float("nan")), dict(dtype=2), dict(st=62), dict(cu=None), dict(Hq=0),
                dict(Tq=-1)):
        assert attn(**bad) == -22, bad
    assert attn(D=136) == -95 and attn(Tq=1 << 30, Hq=4) == -95 and attn(Tq=0) == 0
    assert lib.sam3_seq_attn_bwd(*([p, 64, 64] * 4), p, p, p, p, p, p, p, 8, 8, 1, 4, 2, 64, 8, 8, 1, 0.1, 0, None, 0, None) == -12


def test_strides_that_the_attention_kernels_cannot_follow_are_refused():
    import ctypes
    lib, p, far = _ffi.load(), ctypes.c_void_p(64), 1 << 22

    def call(qs=(64, 64), ks=(64, 64), vs=(64, 64), gs=(64, 64), hk=2, back=True):
        if back:
            return lib.sam3_seq_attn_bwd(p, *qs, p, *ks, p, *vs, p, *gs, p, p, p, p, p, p, p, 8, 8, 1, 4, hk, 64, 8, 8, 1, 0.1, 0, p, 1 << 20, None)
        return lib.sam3_seq_attn_fwd(p, *qs, p, *ks, p, *vs, p, p, None, p, None, None, 8, 8, 1, 4, hk, 64, 8, 8, 1, 0.1, 0, None, 0, None)
    for back in (False, True):
        for bad in (dict(qs=(far, 64)), dict(qs=(64, far)), dict(ks=(far, 64)), dict(vs=(far, 64)), dict(qs=(far, 64), hk=4)) + ((dict(gs=(far, 64)), dict(gs=(64, far))) if back else ()):
            assert call(back=back, **bad) == -95 and "2^22" in lib.sam3_seq_last_error().decode(), bad
        for bad in (dict(qs=(-64, 64)), dict(ks=(64, -64)), dict(vs=(64, 60))):
            assert call(back=back, **bad) == -22, bad
    with pytest.raises(ValueError, match="do not fit"):
        sequence._rotation_table((0,) * 256 + (8,), 10000.0, "shared", 64)
    assert list(sequence._rotation_table((0,) * 255 + (8,), 10000.0, "shared", 64)[1]) == [255] * 8


def test_calls_are_refused_before_they_reach_the_gpu():
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(LoRAKernelError, match="AMD GPU"):
        sequence.rms_norm(x, w)
    with pytest.raises(LoRAKernelError, match="bfloat16 or float32"):
        sequence.rms_norm(x.half(), w.half())
    with pytest.raises(LoRAKernelError, match="AMD GPU"):
        sequence.rotary_axes(torch.zeros(2, 3, 64), None, torch.zeros(1, 2, dtype=torch.int32), (32,))
    q = torch.zeros(4, 2, 64)
    with pytest.raises(LoRAKernelError, match="AMD GPU"):
        sequence.packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(TypeError):
        sequence.rms_norm([1.0], w)


@pytest.mark.gpu
def test_arguments_are_checked():
    dev = "cuda"
    x, w = torch.zeros(4, 64, device=dev), torch.ones(64, device=dev)
    for bad in (lambda: sequence.rms_norm(x, w[:32]), lambda: sequence.rms_norm(x[:, :60], w[:60]), lambda: sequence.rms_norm(x, w.bfloat16()),
                lambda: sequence.rms_norm(x, w, residual=x[:2]), lambda: sequence.rms_norm(x, w, eps=-1.0), lambda: sequence.rms_norm(x, w.cpu()),
                lambda: sequence.rms_norm_q8(x, w, group=16), lambda: sequence.rms_norm_q8(x, w, group=128), lambda: sequence.rms_norm_q8(x, w, fmt=7),
                lambda: sequence.rms_norm_q8(x.clone().requires_grad_(True), w)):
        with pytest.raises(ValueError):
            bad()
    q, k = torch.zeros(4, 4, 64, device=dev), torch.zeros(4, 2, 64, device=dev)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    for bad in (lambda: sequence.rotary_axes(q, k, pos, (33,)), lambda: sequence.rotary_axes(q, k, pos, ()), lambda: sequence.rotary_axes(q, k, pos, (16, 16)),
                lambda: sequence.rotary_axes(q, k[:3], pos, (32,)), lambda: sequence.rotary_axes(q, k, pos, (32,), pairing="x"),
                lambda: sequence.rotary_axes(q, k, pos, (32,), spectrum="x"), lambda: sequence.rotary_axes(q, k, pos, (32,), theta=0.0),
                lambda: sequence.rotary_axes(q, k, pos.cpu(), (32,)), lambda: sequence.rotary_axes(q[..., :60], k[..., :60], pos, (16,))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        sequence.rotary_axes(q, k, pos.double(), (32,))
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    for bad in (lambda: sequence.packed_attention(q, k[:3], k[:3], cu), lambda: sequence.packed_attention(q, k, k[..., :32], cu),
                lambda: sequence.packed_attention(q[:, :3], k, k, cu), lambda: sequence.packed_attention(q, k, k, cu, cu[:1]),
                lambda: sequence.packed_attention(q, k, k, cu.cpu()), lambda: sequence.packed_attention(q, k, k, cu, scale=0.0),
                lambda: sequence.packed_attention(q, k, k, cu, max_q=-1), lambda: sequence.packed_attention(q, k, k, cu, len_k=cu),
                lambda: sequence.packed_attention(q.clone().requires_grad_(True), k, k, cu, len_k=cu[1:]),
                lambda: sequence.packed_attention(q.bfloat16(), k, k, cu)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sequence.packed_attention(q, k, k, cu.long()), lambda: sequence.packed_attention(q, k, k, [0, 4])):
        with pytest.raises(TypeError):
            bad()


# ----------------------------------------------------------------------------------------------------------- RMS norm
def norm_ref(x, w, r, eps, gy=None, gh=None):
    h = x if r is None else x + r
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = h * rstd
    out = dict(h=h, y=xhat * w, xhat=xhat, rstd=rstd)
    if gy is not None:
        u = gy * w
        out["mean"] = (u * xhat).mean(-1, keepdim=True)
        out["gx"] = rstd * (u - xhat * out["mean"]) + (0 if gh is None else gh)
        out["gw"] = (gy * xhat).sum(0)
        out["u"] = u
    return out


# fp32 operations on the way to y: the sum of squares (a lane adds at most 64 of them, then 8 levels), the mean, eps, the root (2),
# the products (3), half of the sum's part reaching y through the root
NORM_OPS = 48


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 8), (1, 1024), (3, 64), (37, 72), (130, 128), (65, 264), (5, 512), (9, 520), (33, 1024), (7, 2040),
                                        (5, 4096), (3, 4104), (2, 6152), (3, 16384), (2050, 96)])
def test_rms_norm_and_gradients(rows, width, residual, dtype):
    g = gen(rows * 7 + width)
    gain = torch.exp(0.5 * torch.randn(width, generator=g))
    x = (torch.randn(rows, width, generator=g) * gain).to(dtype).double()
    r = (torch.randn(rows, width, generator=g) * gain * 2).to(dtype).double() if residual else None
    w = rand(g, width, dtype=dtype, scale=0.3) + 1
    w = w.to(dtype).double()
    gy, gh = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype) if residual else None
    ref = norm_ref(x, w, r, 1e-6, gy, gh)
    u = unit(dtype)
    dev = lambda t: None if t is None else t.to("cuda", dtype)      # noqa: E731
    xs = dev(x).requires_grad_(True)
    rs = dev(r).requires_grad_(True) if residual else None
    ws = dev(w).requires_grad_(True)
    got = sequence.rms_norm(xs, ws, residual=rs)
    y = got[0] if residual else got
    assert y.dtype == dtype
    close(y, ref["y"], (u + NORM_OPS * F) * ref["y"].abs(), "y")
    if residual:
        close(got[1], ref["h"], (u + F) * ref["h"].abs(), "h")
        grads = torch.autograd.grad(got, (xs, rs, ws), (dev(gy), dev(gh)))
        assert torch.equal(grads[0], grads[1])
    else:
        grads = torch.autograd.grad(y, (xs, ws), dev(gy))
    # the saved stream is rounded once (u, with a residual): it reaches xhat, and through the mean of u xhat the result
    us = u if residual else 0.0
    absmean = (ref["u"] * ref["xhat"]).abs().mean(-1, keepdim=True)
    tol = ref["rstd"] * (2 * NORM_OPS * F * (ref["u"].abs() + ref["xhat"].abs() * absmean) + 2 * us * ref["xhat"].abs() * absmean)
    close(grads[0], ref["gx"], tol + (u + 2 * F) * ref["gx"].abs() + 2 * F * (0 if gh is None else gh.abs()), "gx")
    sums = (gy * ref["xhat"]).abs().sum(0)
    close(grads[-1], ref["gw"], u * ref["gw"].abs() + (us + (rows + NORM_OPS) * F) * sums, "gw")
    with torch.no_grad():       # without a gradient: the same kernel
        again = sequence.rms_norm(dev(x), dev(w), residual=dev(r))
    assert torch.equal(again[0] if residual else again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(1, 8), (37, 72), (300, 1024), (40, 2056)])
def test_rms_norm_gradients_know_two_bits_more_than_the_stream(rows, width):
    """bf16 with a residual: the two bits leave at most 3/16 of a last place of h, which is 2 u at most: 3/8 u where the rounded h has u."""
    dtype, g = torch.bfloat16, gen(rows + width)
    x, r = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype, scale=0.37)
    x[0, :3], r[0, :3] = 0.0, torch.tensor([0.0, -0.0, 2.0 ** -120])        # nothing, and next to nothing
    x[-1, 4:8], r[-1, 4:8] = torch.tensor([1.0, -1.0, 1.0, 2.0]).double(), torch.tensor([2.0 ** -8, 2.0 ** -8, -2.0 ** -9, -2.0 ** -8]).double()    # halves and quarters of a place
    w, gy, gh = (rand(g, width, dtype=dtype, scale=0.3) + 1).to(dtype).double(), rand(g, rows, width, dtype=dtype), torch.zeros(rows, width, dtype=torch.double)
    ref = norm_ref(x, w, r, 1e-6, gy, gh)
    leaves = [t.to("cuda", dtype).requires_grad_(True) for t in (x, r, w)]
    got = sequence.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    grads = torch.autograd.grad(got, leaves, (gy.to("cuda", dtype), gh.to("cuda", dtype)))
    u = unit(dtype)
    us = 3 / 8 * u
    absmean = (ref["u"] * ref["xhat"]).abs().mean(-1, keepdim=True)
    tol = ref["rstd"] * (2 * NORM_OPS * F * (ref["u"].abs() + ref["xhat"].abs() * absmean) + 2 * us * ref["xhat"].abs() * absmean)
    close(grads[0], ref["gx"], tol + (u + 2 * F) * ref["gx"].abs(), "gx")
    close(grads[2], ref["gw"], u * ref["gw"].abs() + (us + (rows + NORM_OPS) * F) * (gy * ref["xhat"]).abs().sum(0), "gw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("fmt", [sequence.FP8_E4M3, sequence.FP8_E5M2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,width,group", [(1, 32, 32), (3, 1024, 0), (17, 128, 128), (33, 64, 64), (5, 1056, 32), (2, 4224, 128), (4, 8192, 0), (129, 512, 64)])
def test_rms_norm_q8(rows, width, group, fmt, dtype):
    g = gen(rows + width + group)
    x, r = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype, scale=3)
    if rows > 2:
        x[1], r[1] = 0, 0                       # a row without content
    w = rand(g, width, dtype=dtype)
    ref = norm_ref(x, w, r, 1e-6)
    image, scales, h = sequence.rms_norm_q8(x.to("cuda", dtype), w.to("cuda", dtype), residual=r.to("cuda", dtype), group=group, fmt=fmt)
    close(h, ref["h"], (unit(dtype) + F) * ref["h"].abs(), "h")
    parts = ref["y"].reshape(rows, -1, group or width)
    top, half, tiny = (448.0, 2.0 ** -4, 2.0 ** -10) if fmt == sequence.FP8_E4M3 else (57344.0, 2.0 ** -3, 2.0 ** -17)
    want = parts.abs().amax(-1).clamp(min=2.0 ** -24) / top
    assert image.dtype == (torch.float8_e4m3fn if fmt == sequence.FP8_E4M3 else torch.float8_e5m2) and scales.dtype == torch.float32
    close(scales, want, (NORM_OPS + 2) * F * want, "scales")
    # against the scale that came out: one rounding to 8 bits (half a step of the value, or of the smallest exponent), the fp32 errors before it
    value = parts / scales.cpu().double()[..., None]
    back = image.cpu().float().double().reshape(parts.shape)
    close(back, value, torch.clamp(half * value.abs(), min=tiny) * (1 + 2.0 ** -12) + (NORM_OPS + 4) * F * value.abs(), "image")
    alone = sequence.rms_norm_q8(x.to("cuda", dtype), w.to("cuda", dtype), group=group, fmt=fmt)
    assert len(alone) == 2


@pytest.mark.gpu
def test_rms_norm_rows_of_a_wider_tensor_other_shapes_and_no_rows():
    g = gen(3)
    big = torch.randn(6, 5, 3 * 256, generator=g).to("cuda", torch.bfloat16)
    x, r, w = big[..., 256:512], big[..., 512:], torch.ones(256, device="cuda", dtype=torch.bfloat16)
    y, h = sequence.rms_norm(x, w, residual=r)
    y2, h2 = sequence.rms_norm(x.contiguous(), w, residual=r.contiguous())
    assert y.shape == x.shape and torch.equal(y, y2) and torch.equal(h, h2)
    odd = torch.randn(7 * 64 + 1, generator=g).to("cuda", torch.bfloat16)[1:].view(7, 64)       # not 16-byte aligned
    assert torch.equal(sequence.rms_norm(odd, w[:64]), sequence.rms_norm(odd.clone(), w[:64]))
    assert torch.equal(sequence.rms_norm(x[0, 0], w), y.new_tensor(sequence.rms_norm(x[:1, :1], w).tolist())[0, 0])
    empty = torch.empty(0, 64, device="cuda", requires_grad=True)
    wt = torch.ones(64, device="cuda", requires_grad=True)
    out = sequence.rms_norm(empty, wt)
    gx, gw = torch.autograd.grad(out, (empty, wt), torch.empty_like(out))
    assert out.shape == (0, 64) and gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(gw))
    spread = torch.randn(64, generator=g).cuda().expand(5, 64).requires_grad_(True)             # a broadcast input
    out = sequence.rms_norm(spread, wt)
    assert torch.equal(out, sequence.rms_norm(spread.contiguous(), wt))


@pytest.mark.gpu
def test_rms_norm_partial_gradients():
    g = gen(4)
    x, r, w = (torch.randn(*s, generator=g).cuda() for s in ((9, 64), (9, 64), (64,)))
    gy, gh = torch.randn(9, 64, generator=g).cuda(), torch.randn(9, 64, generator=g).cuda()
    xs = x.clone().requires_grad_(True)
    y, h = sequence.rms_norm(xs, w, residual=r)
    full = torch.autograd.grad((y, h), xs, (gy, gh), retain_graph=True)[0]
    only_y = torch.autograd.grad(y, xs, gy, retain_graph=True)[0]
    only_h = torch.autograd.grad(h, xs, gh)[0]
    assert torch.equal(only_h, gh)
    assert (full - (only_y + gh)).abs().max() <= 4 * F * (only_y.abs() + gh.abs()).max()
    ws = w.clone().requires_grad_(True)
    y, h = sequence.rms_norm(x, ws, residual=r)
    ref = norm_ref(x.cpu().double(), w.cpu().double(), r.cpu().double(), 1e-6, gy.cpu().double())
    close(torch.autograd.grad(y, ws, gy)[0], ref["gw"], (9 + NORM_OPS) * F * (gy.cpu().double() * ref["xhat"]).abs().sum(0), "gw")


@pytest.mark.gpu
def test_rms_norm_keeps_rows_apart_and_non_finite_rows_to_themselves():
    x = torch.randn(70, 128, generator=gen(5)).cuda()
    w = torch.ones(128, device="cuda")
    good = sequence.rms_norm_q8(x, w)
    bad = x.clone()
    bad[3, 5], bad[40, 0] = float("nan"), float("inf")
    image, scales = sequence.rms_norm_q8(bad, w)
    keep = torch.ones(70, dtype=torch.bool)
    keep[[3, 40]] = False
    assert torch.equal(image.view(torch.uint8)[keep], good[0].view(torch.uint8)[keep]) and torch.equal(scales[keep], good[1][keep])
    assert torch.isnan(image.float()[3]).all() and torch.isnan(scales[3]).all() and not torch.isfinite(image.float()[40, 0])


# --------------------------------------------------------------------------------------------------- rotary positions
def rope_ref(x, pos, sections, theta, pairing, spectrum, sign=1.0):
    n = sum(sections)
    axis = [a for a, m in enumerate(sections) for _ in range(m)]
    rate = [theta ** (-i / n) for i in range(n)] if spectrum == "shared" else [theta ** (-i / m) for m in sections for i in range(m)]
    angle = pos.double()[axis].movedim(0, -1) * torch.tensor(rate, dtype=torch.float64) * sign
    cos, sin = angle.cos()[..., None, :], angle.sin()[..., None, :]
    first = torch.arange(n) * 2 if pairing == "adjacent" else torch.arange(n)
    second = first + 1 if pairing == "adjacent" else first + n
    out, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size


# cos and sin: the fraction of a turn is rounded to fp32 (2^-25 of half a turn: an angle of 2 pi 2^-26), the functions are good to 2 ulp;
# then two products and a sum
ROPE_OPS = 2 * math.pi / 4 + 4 + 3
ROPE = [  # heads, kv heads, D, sections, pairing, spectrum
    (1, 1, 8, (4,), "adjacent", "shared"), (3, 1, 64, (32,), "halves", "shared"), (4, 2, 64, (8, 12, 12), "adjacent", "per_axis"),
    (16, 4, 128, (16, 24, 24), "halves", "shared"), (2, 2, 96, (7, 0, 6), "halves", "shared"), (5, 1, 40, (3, 2), "adjacent", "per_axis"),
    (2, 1, 256, (32, 32, 32, 32), "halves", "per_axis"), (8, 8, 64, (16, 8), "halves", "per_axis"), (7, 7, 32, (5, 4, 3), "halves", "shared")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("tokens,kind", [(1, "i32"), (7, "i64"), (65, "f32"), (1030, "i32"), (4099, "f32")])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(str(v) for v in c))
def test_rotary_axes_and_gradients(case, tokens, kind, dtype):
    hq, hk, d, sections, pairing, spectrum = case
    if tokens * hq * d > 2_000_000:
        tokens = 4099 // 8
    g = gen(tokens + d)
    qkv = rand(g, tokens, hq + 2 * hk, d, dtype=dtype)
    far = torch.randint(-(1 << 20), 1 << 20, (len(sections), tokens), generator=g)
    pos = far.int() if kind == "i32" else far * 1024 if kind == "i64" else far.float() / 64
    fused = qkv.to("cuda", dtype).requires_grad_(True)
    q, k = fused[:, :hq], fused[:, hq:hq + hk]
    got = sequence.rotary_axes(q, k, pos.cuda(), sections, theta=10000.0, pairing=pairing, spectrum=spectrum)
    go = [rand(g, tokens, n, d, dtype=dtype) for n in (hq, hk)]
    grad = torch.autograd.grad(got, fused, [t.to("cuda", dtype) for t in go])[0]
    u = unit(dtype)
    for out, lo, n in ((got[0], 0, hq), (got[1], hq, hk)):
        want, size = rope_ref(qkv[:, lo:lo + n], pos, sections, 10000.0, pairing, spectrum)
        close(out, want, u * want.abs() + ROPE_OPS * F * size, "out")
    for t, lo, n in ((go[0], 0, hq), (go[1], hq, hk)):
        want, size = rope_ref(t, pos, sections, 10000.0, pairing, spectrum, -1.0)
        close(grad[:, lo:lo + n], want, u * want.abs() + ROPE_OPS * F * size, "grad")
    assert torch.equal(grad[:, hq + hk:], torch.zeros_like(grad[:, hq + hk:]))
    alone = sequence.rotary_axes(q.detach(), None, pos.cuda(), sections, theta=10000.0, pairing=pairing, spectrum=spectrum)
    assert torch.equal(alone, got[0])


@pytest.mark.gpu
def test_rotary_axes_matches_the_trunks_tables():
    """The trunk's 2-D tables and kernel are one setting of the general operator."""
    from sam3_lora_amd import vit
    att = vit.Attention(128, 2, True, (6, 5), rope_theta=10000.0).cuda()
    qkv = torch.randn(2, 30, 3, 2, 64, generator=gen(8)).cuda()
    cos, sin = att._cos_sin(qkv.device)
    q, k, _ = vit._QKVRope.apply(qkv.reshape(60, 384), cos, sin, 2, 30, 2, 64)
    t = torch.arange(30, device="cuda")
    pos = torch.stack([t % 6, t // 6]).int()[:, None].expand(2, 2, 30)
    q2, k2 = sequence.rotary_axes(qkv[:, :, 0], qkv[:, :, 1], pos, (16, 16), spectrum="per_axis")
    # both round cos and sin to fp32; the table's angles are fp32 products (up to 6 of 2^-24 of an angle up to 5)
    assert (q - q2).abs().max() <= 40 * F * 8 and (k - k2).abs().max() <= 40 * F * 8


@pytest.mark.gpu
def test_rotary_axes_edges():
    q = torch.randn(5, 2, 64, generator=gen(9)).cuda()
    pos = torch.arange(5, device="cuda")[None]
    assert torch.equal(sequence.rotary_axes(q, None, torch.zeros_like(pos), (32,)), q)
    q2 = q.clone()
    q2[2, 1, 40:] = float("inf")                # behind the turned part: copied as it is
    out = sequence.rotary_axes(q2, None, pos, (19,))
    assert torch.equal(out[..., 38:], q2[..., 38:]) and torch.isfinite(out[..., :38]).all()
    out = sequence.rotary_axes(q2, None, pos, (19,), pairing="halves")
    assert torch.equal(out[..., 38:], q2[..., 38:]) and torch.isfinite(out[..., :38]).all()
    assert sequence.rotary_axes(q[:0], q[:0], pos[:, :0], (32,))[0].shape == (0, 2, 64)
    odd = torch.randn(5 * 2 * 64 + 1, generator=gen(10)).cuda()[1:].view(5, 2, 64)
    assert torch.equal(sequence.rotary_axes(odd, None, pos, (32,)), sequence.rotary_axes(odd.clone(), None, pos, (32,)))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(sequence.rotary_axes(heads_first, None, pos, (32,)), sequence.rotary_axes(q, None, pos, (32,)))
    qs, ks = q.clone().requires_grad_(True), q.clone().requires_grad_(True)
    a, b = sequence.rotary_axes(qs, ks, pos, (32,))
    assert torch.equal(torch.autograd.grad(b.sum(), ks, retain_graph=True)[0], torch.autograd.grad(a.sum(), qs)[0])


# ---------------------------------------------------------------------------------------------------------- attention
def attn_ref(q, k, v, lq, lk, causal, scale, u, go=None, len_k=None, uw=None):
    """Results and error bounds in 64 bits: the bounds follow the roundings named at each line.  uw: of a weight, or of dS (u)."""
    uw = u if uw is None else uw
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    r = {n: torch.zeros_like(t) for n, t in (("o", q), ("to", q), ("gq", q), ("tgq", q), ("gk", k), ("tgk", k), ("gv", v), ("tgv", v))}
    r["lse"] = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    r["tlse"] = torch.zeros(q.shape[:2], dtype=torch.float64)
    a = b = 0
    for i, (m, n) in enumerate(zip(lq, lk)):
        nn = n if len_k is None else len_k[i]
        for h in range(hq):
            kh = h // (hq // hk)
            Q, K, V = q[a:a + m, h], k[b:b + nn, kh], v[b:b + nn, kh]
            seen = torch.ones(m, nn, dtype=torch.bool).tril(nn - m) if causal else torch.ones(m, nn, dtype=torch.bool)
            s = (Q @ K.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0.0) if nn else torch.zeros(m, 0, dtype=torch.float64)
            o = p @ V
            # scores: a sum of d products, scale log2(e) and the maximum joined in one fused step, the exponential good to 2 ulp; both
            # the row's sum and the weight carry it
            es = ((d + 6) * F * (Q.abs() @ K.abs().T) * scale + 6 * F * s.abs().masked_fill(~seen, 0.0) + 4 * F).masked_fill(~seen, 0.0)
            worst = es.amax(1, keepdim=True) if nn else es.new_zeros(m, 1)
            ep = es + worst + (nn + 16) * F            # relative, of a weight; the sum of nn terms and its rescalings
            to = ((ep + uw) * p) @ V.abs() + (nn + 16) * F * (p @ V.abs()) + u * o.abs()      # the weight's rounding, the result's
            r["o"][a:a + m, h], r["to"][a:a + m, h] = o, to
            if nn:
                r["lse"][a:a + m, h] = torch.logsumexp(s, 1)
                fin = torch.isfinite(r["lse"][a:a + m, h])
                r["tlse"][a:a + m, h] = torch.where(fin, worst[:, 0] + (nn + 16) * F + 4 * F * r["lse"][a:a + m, h].abs().masked_fill(~fin, 0.0), 0.0)
            if go is not None:
                G = go[a:a + m, h]
                dp = G @ V.T
                delta = (G * o).sum(1, keepdim=True)
                ds = p * (dp - delta)
                # the forward's rounded result in delta, its sum of d products, and those of dp
                ed = (G.abs() * to).sum(1, keepdim=True) + (d + 2) * F * (G.abs() * o.abs()).sum(1, keepdim=True)
                ep2 = 2 * ep + 4 * F                   # weights recomputed from the stored fp32 lse
                eds = p * ((d + 2) * F * (G.abs() @ V.abs().T) + ed) + (ep2 + 4 * F) * ds.abs() + uw * ds.abs()
                r["gq"][a:a + m, h] = ds @ K * scale
                r["tgq"][a:a + m, h] = (eds @ K.abs() + (nn + 2) * F * (ds.abs() @ K.abs())) * scale + (u + 2 * F) * r["gq"][a:a + m, h].abs()
                rows = m * (hq // hk)
                r["gk"][b:b + nn, kh] += ds.T @ Q * scale
                r["tgk"][b:b + nn, kh] += (eds.T @ Q.abs() + (rows + 2) * F * (ds.abs().T @ Q.abs())) * scale
                r["gv"][b:b + nn, kh] += p.T @ G
                r["tgv"][b:b + nn, kh] += ((ep2 + uw) * p).T @ G.abs() + (rows + 2) * F * (p.T @ G.abs())
        a, b = a + m, b + n
    r["tgk"] += (u + 2 * F) * r["gk"].abs()
    r["tgv"] += (u + 2 * F) * r["gv"].abs()
    return r


def ends(lengths, dev="cuda"):
    return torch.tensor([0] + list(lengths)).cumsum(0).int().to(dev)


def check_attention(lq, lk, hq, hk, d, causal, dtype, seed=0, scale=None, train=True, hints=True, qscale=1.5):
    g = gen(seed)
    q = rand(g, sum(lq), hq, d, dtype=dtype, scale=qscale)
    k, v = rand(g, sum(lk), hk, d, dtype=dtype), rand(g, sum(lk), hk, d, dtype=dtype)
    go = rand(g, sum(lq), hq, d, dtype=dtype)
    ref = attn_ref(q, k, v, lq, lk, causal, scale or d ** -0.5, unit(dtype), go if train else None)
    qs, ks, vs = (t.to("cuda", dtype).requires_grad_(train) for t in (q, k, v))
    how = dict(max_q=max(lq, default=0), max_k=max(lk, default=0)) if hints else {}
    out, lse = sequence.packed_attention(qs, ks, vs, ends(lq), ends(lk), causal=causal, scale=scale, return_lse=True, **how)
    close(out, ref["o"], ref["to"], "out")
    fin = torch.isfinite(ref["lse"])
    assert torch.equal(torch.isfinite(lse.cpu()), fin) and (lse.cpu()[~fin] == -math.inf).all()
    close(lse.cpu()[fin], ref["lse"][fin], ref["tlse"][fin], "lse")
    if train:
        grads = torch.autograd.grad(out, (qs, ks, vs), go.to("cuda", dtype))
        for n, t in zip(("gq", "gk", "gv"), grads):
            close(t, ref[n], ref["t" + n], n)
        again = torch.autograd.grad(sequence.packed_attention(qs, ks, vs, ends(lq), ends(lk), causal=causal, scale=scale, **how), (qs, ks, vs), go.to("cuda", dtype))
        assert all(torch.equal(a, b) for a, b in zip(grads, again))


ATTN = [  # query lengths, key lengths, heads, kv heads, D, causal
    ([1], [1], 1, 1, 8, True), ([2, 1, 5], [2, 1, 5], 2, 1, 32, True), ([33], [33], 1, 1, 64, True), ([64, 64], [64, 64], 4, 4, 64, True),
    ([65, 1, 31], [65, 1, 31], 4, 2, 64, True), ([129], [129], 2, 1, 128, True), ([200, 3], [200, 3], 3, 3, 40, True),
    ([130, 70], [130, 70], 6, 1, 96, True), ([17, 90], [17, 90], 7, 1, 128, True), ([5, 0, 9], [5, 0, 9], 2, 2, 64, True),
    ([0, 0], [0, 0], 2, 1, 64, True), ([4], [300], 4, 2, 64, True), ([40, 3], [10, 3], 2, 1, 64, True), ([10, 5], [0, 7], 2, 1, 64, True),
    ([100], [35], 2, 2, 128, True), ([1, 1, 1], [1, 257, 64], 8, 2, 128, True), ([3, 2], [1000, 130], 4, 1, 64, True),
    ([70], [70], 2, 2, 64, False), ([1], [200], 2, 1, 64, False), ([150, 20], [33, 97], 4, 2, 32, False), ([64], [128], 2, 1, 128, False),
    ([12, 0, 4], [0, 5, 9], 2, 1, 24, False), ([260], [260], 2, 1, 64, True), ([300], [300], 1, 1, 128, False),
    ([9, 30], [9, 30], 40, 1, 64, True), ([5, 3], [70, 3], 64, 1, 32, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(v).replace(" ", "") for v in c))
def test_packed_attention_and_gradients(case, dtype):
    check_attention(*case, dtype, seed=len(case[0]) + case[4])


MANY = [  # as above, often enough for the tiles of 128 rows and keys (more than 256 of them over the pairs)
    ([130, 70, 1, 0, 65], 2, 2, 64, True, 40), ([200, 3], 4, 2, 128, True, 50), ([33, 140], 3, 1, 32, True, 150), ([90], 7, 1, 64, True, 260),
    ([150, 64], 6, 2, 96, False, 60), ([129], 10, 2, 128, False, 70), ([40, 31], 5, 1, 128, True, 140)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(str(v).replace(" ", "") for v in c))
def test_packed_attention_many_sequences(case, dtype):
    lens, hq, hk, d, causal, times = case
    check_attention(lens * times, lens * times, hq, hk, d, causal, dtype, seed=d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_many_sequences_of_other_key_lengths(d, dtype):
    lq, lk = [40, 100, 7, 0, 130] * 30, [140, 60, 7, 9, 200] * 30
    for causal in (True, False):
        check_attention(lq, lk, 4, 2, d, causal, dtype, seed=d, hints=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
def test_packed_attention_hints_and_scale(dtype):
    check_attention([150, 40], [150, 40], 4, 2, 64, True, dtype, hints=False)
    check_attention([50], [50], 2, 2, 64, True, dtype, scale=0.5)
    # a hint that is too small costs time, not the result (it may choose another order of the sums)
    g = gen(1)
    q, k = rand(g, 300, 2, 64, dtype=dtype), rand(g, 300, 2, 64, dtype=dtype)
    ref = attn_ref(q, k, k, [300], [300], True, 0.125, unit(dtype), q)
    leaves = [t.to("cuda", dtype).requires_grad_(True) for t in (q, k, k)]
    for hint in (dict(max_q=1, max_k=300), dict(max_q=1, max_k=1), dict(max_q=0, max_k=0), {}):
        out = sequence.packed_attention(*leaves, ends([300]), **hint)
        close(out, ref["o"], ref["to"], "out")
        for n, t in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, q.to("cuda", dtype))):
            close(t, ref[n], ref["t" + n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("lq,lk,hq,hk,d", [([1, 1, 1], [300, 1, 5000], 8, 2, 128), ([1] * 5, [129, 2000, 31, 0, 257], 4, 1, 64), ([3, 1], [1500, 700], 4, 4, 32),
                                           ([40], [3000], 4, 2, 64), ([70, 9], [1100, 2050], 2, 2, 96), ([8], [129], 4, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_few_rows_over_many_keys(lq, lk, hq, hk, d, causal, dtype):
    check_attention(lq, lk, hq, hk, d, causal, dtype, seed=d)
    check_attention(lq, lk, hq, hk, d, causal, dtype, seed=d + 1, train=False, hints=False)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,hq,hk,d", [([1, 1, 1], [300, 1, 2000], 8, 2, 64), ([20, 3, 31], [20, 3, 31], 4, 4, 64), ([2, 7], [60, 9], 4, 2, 128),
                                           ([30], [30], 1, 1, 32), ([1], [5000], 1, 1, 128)])
def test_packed_attention_of_few_rows_keeps_16_bits_of_the_weights(lq, lk, hq, hk, d):
    """bf16, one tile of rows or one block of the other side: weights and dS go into the products as two roundings to bf16, u^2 off."""
    dtype, g = torch.bfloat16, gen(23)
    q, go = rand(g, sum(lq), hq, d, dtype=dtype, scale=1.5), rand(g, sum(lq), hq, d, dtype=dtype)
    k, v = rand(g, sum(lk), hk, d, dtype=dtype), rand(g, sum(lk), hk, d, dtype=dtype)
    u = unit(dtype)
    ref = attn_ref(q, k, v, lq, lk, True, d ** -0.5, u, go, uw=u * u)
    leaves = [t.to("cuda", dtype).requires_grad_(True) for t in (q, k, v)]
    out = sequence.packed_attention(*leaves, ends(lq), ends(lk), max_q=max(lq), max_k=max(lk))
    close(out, ref["o"], ref["to"], "out")
    for n, t in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, go.to("cuda", dtype))):
        close(t, ref[n], ref["t" + n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("nq", [1, 3, 50])
def test_packed_attention_over_caches_with_room(nq, dtype):
    """Caches [B, room, 2, Hk, D], of which len_k rows are in use; what lies behind them is not touched, NaN or not."""
    g = gen(nq)
    B, room, hq, hk, d = 4, 700, 4, 2, 64
    used = [700, 333, 0, nq]
    cache = rand(g, B, room, 2, hk, d, dtype=dtype).to("cuda", dtype)
    for b, n in enumerate(used):
        cache[b, n:] = float("nan")
    q = rand(g, B * nq, hq, d, dtype=dtype)
    flat = cache.view(B * room, 2, hk, d)
    cu_q, cu_k = ends([nq] * B), ends([room] * B)
    out = sequence.packed_attention(q.to("cuda", dtype), flat[:, 0], flat[:, 1], cu_q, cu_k, max_q=nq, max_k=room,
                                    len_k=torch.tensor(used, dtype=torch.int32, device="cuda"))
    clean = torch.nan_to_num(cache, nan=0.0).cpu().double().view(B * room, 2, hk, d)
    ref = attn_ref(q, clean[:, 0], clean[:, 1], [nq] * B, [room] * B, True, d ** -0.5, unit(dtype), len_k=used)
    close(out, ref["o"], ref["to"], "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
def test_packed_attention_rows_of_no_sequence_and_bad_bounds(dtype):
    g = gen(11)
    q, k = rand(g, 90, 4, 64, dtype=dtype), rand(g, 70, 2, 64, dtype=dtype)
    qs, ks, vs = (t.to("cuda", dtype).requires_grad_(True) for t in (q, k, k))
    cu_q, cu_k = torch.tensor([5, 25, 61], dtype=torch.int32, device="cuda"), torch.tensor([3, 23, 60], dtype=torch.int32, device="cuda")
    out, lse = sequence.packed_attention(qs, ks, vs, cu_q, cu_k, return_lse=True)
    go = rand(g, 90, 4, 64, dtype=dtype)
    grads = torch.autograd.grad(out, (qs, ks, vs), go.to("cuda", dtype))
    ref = attn_ref(q[5:61], k[3:60], k[3:60], [20, 36], [20, 37], True, 0.125, unit(dtype), go[5:61])
    close(out[5:61], ref["o"], ref["to"], "out")
    for t, n, (a, b) in zip(grads, ("gq", "gk", "gv"), ((5, 61), (3, 60), (3, 60))):
        close(t[a:b], ref[n], ref["t" + n], n)
        assert not t[:a].any() and not t[b:].any()
    assert not out[:5].any() and not out[61:].any() and (lse[:5] == -math.inf).all() and (lse[61:] == -math.inf).all()
    # bounds outside the tensors or in no order are clamped: the call stays inside its tensors
    wild = torch.tensor([-7, 1000, 3, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out = sequence.packed_attention(qs, ks, vs, wild, wild)
    assert all(t.shape == u.shape for t, u in zip(torch.autograd.grad(out, (qs, ks, vs), go.to("cuda", dtype)), (qs, ks, vs)))
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not sequence.packed_attention(qs, ks, vs, none, none).any()
    empty = sequence.packed_attention(qs[:0], ks, vs, ends([0]), ends([70]))
    assert empty.shape == (0, 4, 64)
    gk = torch.autograd.grad(empty, ks, empty)[0]
    assert not gk.any()
    out = sequence.packed_attention(qs, ks[:0], vs[:0], ends([90]), ends([0]))
    assert not out.any() and not torch.autograd.grad(out, qs, go.to("cuda", dtype))[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("n,hq,hk,d", [(100, 2, 1, 64), (200, 4, 4, 128), (300, 3, 1, 32)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("others", [0, 300])
def test_packed_attention_what_a_query_does_not_see_stays_out(others, value, n, hq, hk, d, dtype):
    """A token that is not finite spoils the results that depend on it and no others, forward and backward; with 300 more sequences the
    kernels for many tiles run."""
    g = gen(n)
    total = n + 16 * others
    q, k, v, go = (rand(g, total, h, d, dtype=dtype).to("cuda", dtype) for h in (hq, hk, hk, hq))
    cu = ends([n] + [16] * others)
    at, el = n // 2 + 3, 5

    def grads(q, k, v, go):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = sequence.packed_attention(*leaves, cu, max_q=n, max_k=n)
        got = (out,) + torch.autograd.grad(out, leaves, go)
        assert all(torch.isfinite(t[n:]).all() for t in got)
        return tuple(t[:n] for t in got)
    good = grads(q, k, v, go)
    bad_v = v.clone()
    bad_v[at, :, el] = value
    out, gq, gk, gv = grads(q, k, bad_v, go)
    assert torch.equal(out[:at], good[0][:at]) and not torch.isfinite(out[at:, :, el]).any()
    rest = [i for i in range(d) if i != el]
    assert torch.equal(out[at:][..., rest], good[0][at:][..., rest])
    if not math.isnan(value):
        assert (out[at:, :, el] == value).all()
    assert torch.equal(gq[:at], good[1][:at]) and not torch.isfinite(gq[at:]).all(-1).any()
    bad_k = k.clone()
    bad_k[at, :, el] = value
    out, gq, gk, gv = grads(q, bad_k, v, go)
    assert torch.equal(out[:at], good[0][:at]) and torch.equal(gq[:at], good[1][:at])
    # a query or an incoming gradient that is not finite reaches the keys that it sees, not the later ones
    for i in (0, 3):
        args = [q, k, v, go]
        args[i] = args[i].clone()
        args[i][at, :, el] = value
        out, gq, gk, gv = grads(*args)
        assert torch.equal(gk[at + 1:], good[2][at + 1:]) and torch.equal(gv[at + 1:], good[3][at + 1:])
        keep = torch.arange(n, device="cuda") != at
        assert torch.equal(out[keep], good[0][keep]) and torch.equal(gq[keep], good[1][keep])
        assert not torch.isfinite(gk[:at + 1]).all(-1).any()


@pytest.mark.gpu
def test_packed_attention_views_of_a_fused_projection_and_shared_inputs():
    g = gen(12)
    qkv = rand(g, 150, 8, 64, dtype=torch.bfloat16).to("cuda", torch.bfloat16)      # 4 + 2 + 2 heads
    cu = ends([100, 50])
    leaf = qkv.clone().requires_grad_(True)
    out = sequence.packed_attention(leaf[:, :4], leaf[:, 4:6], leaf[:, 6:], cu)
    parts = [t.contiguous().requires_grad_(True) for t in (qkv[:, :4], qkv[:, 4:6], qkv[:, 6:])]
    out2 = sequence.packed_attention(*parts, cu)
    assert torch.equal(out, out2)
    go = rand(g, 150, 4, 64, dtype=torch.bfloat16).to("cuda", torch.bfloat16)
    whole = torch.autograd.grad(out, leaf, go.transpose(0, 1).contiguous().transpose(0, 1))[0]      # a gradient with other strides
    assert torch.equal(whole, torch.cat(torch.autograd.grad(out2, parts, go), 1))
    assert torch.equal(torch.autograd.grad(sequence.packed_attention(*parts, cu).sum(), parts[0])[0],       # a broadcast gradient
                       torch.autograd.grad(sequence.packed_attention(*parts, cu), parts[0], torch.ones_like(out))[0])
    one = parts[1].detach().clone().requires_grad_(True)        # keys that are the values too
    got = torch.autograd.grad(sequence.packed_attention(parts[0], one, one, cu), one, go)[0]
    apart = [one.detach().clone().requires_grad_(True) for _ in range(2)]
    gk, gv = torch.autograd.grad(sequence.packed_attention(parts[0], *apart, cu), apart, go)
    assert torch.equal(got, gk + gv)
    odd = torch.randn(150 * 4 * 24 + 3, generator=g).to("cuda", torch.bfloat16)[3:].view(150, 4, 24)      # not aligned
    assert torch.equal(sequence.packed_attention(odd, odd, odd, cu), sequence.packed_attention(odd.clone(), odd.clone(), odd.clone(), cu))
    spread = parts[1].detach()[:, :1].expand(150, 2, 64)        # one key head for both groups, as a broadcast view
    assert torch.equal(sequence.packed_attention(parts[0].detach(), spread, spread, cu),
                       sequence.packed_attention(parts[0].detach(), spread.contiguous(), spread.contiguous(), cu))


@pytest.mark.gpu
def test_one_token_of_a_wider_buffer_has_any_stride():
    """A view of one token is contiguous whatever its stride between tokens, an odd one too."""
    for dtype in DT:
        buf = torch.randn(3, 4 * 64 + 5, generator=gen(21)).to("cuda", dtype)
        row = buf[1, :256].clone().as_strided((1, 4, 64), (261, 64, 1))
        assert row.is_contiguous() and row.stride(0) == 261
        plain = row.clone()
        pos, cu = torch.full((1, 1), 7, device="cuda"), ends([1])
        for a, b in zip(sequence.rotary_axes(row, row, pos, (32,)), sequence.rotary_axes(plain, plain, pos, (32,))):
            assert torch.equal(a, b)
        leaf, want = row.detach().requires_grad_(True), plain.requires_grad_(True)
        go = buf[2, :256].clone().as_strided((1, 4, 64), (261, 64, 1))
        out, ref = sequence.packed_attention(leaf, leaf, leaf, cu), sequence.packed_attention(want, want, want, cu)
        assert torch.equal(out, ref)
        assert torch.equal(torch.autograd.grad(out, leaf, go)[0], torch.autograd.grad(ref, want, go.clone())[0])
        assert torch.equal(sequence.rms_norm(row.as_strided((1, 256), (261, 1)), buf[0, :256].clone()), sequence.rms_norm(plain.detach().view(1, 256), buf[0, :256].clone()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("nq", [1, 5, 200])
def test_packed_attention_heads_of_a_long_buffer_outside(nq, dtype):
    """[heads, tokens, D] buffers seen as [tokens, heads, D]: heads 2^22 elements and more apart, for the cache, q and out's gradient."""
    g = gen(22)
    room, d = (1 << 22) // 64 + 8, 64
    lk = [300, 70]
    cu_q, cu_k = ends([nq, 3]), ends(lk)

    def outside(n, heads):
        return torch.zeros(heads, room, d, device="cuda", dtype=dtype).transpose(0, 1)[:n].copy_(rand(g, n, heads, d, dtype=dtype))
    q, k, v, go = outside(nq + 3, 4), outside(sum(lk), 2), outside(sum(lk), 2), outside(nq + 3, 4)
    assert min(t.stride(1) for t in (q, k, v, go)) > 1 << 22
    far = [t.detach().requires_grad_(True) for t in (q, k, v)]
    near = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    out, ref = sequence.packed_attention(*far, cu_q, cu_k), sequence.packed_attention(*near, cu_q, cu_k)
    assert torch.equal(out, ref)
    for a, b in zip(torch.autograd.grad(out, far, go), torch.autograd.grad(ref, near, go.contiguous())):
        assert torch.equal(a, b)
    alone = [t[:, :2] for t in (q, k, v)]           # one query head to each key head: q is read where it lies
    assert torch.equal(sequence.packed_attention(*alone, cu_q, cu_k), sequence.packed_attention(*(t.contiguous() for t in alone), cu_q, cu_k))
    with torch.no_grad(), pytest.raises(LoRAKernelError, match="2\\^22"):
        apart = torch.zeros((1 << 22) + 2 * d, device="cuda", dtype=dtype).as_strided((2, 2, d), (1 << 22, d, 1))
        sequence.packed_attention(q, apart, apart, cu_q, ends([1, 1]))


@pytest.mark.gpu
def test_packed_attention_cache_rows_beyond_32_bits():
    """Rows so far apart that their offsets in bytes, and in elements, pass 2^32."""
    g = gen(13)
    rows, pitch = 2300, 2_000_000
    big = torch.empty(rows * pitch, device="cuda", dtype=torch.bfloat16)          # 9.2 GB, used in strips
    k = big.as_strided((rows, 1, 64), (pitch, 64, 1))
    v = big.as_strided((rows, 1, 64), (pitch, 64, 1), 64)
    kk, vv = (rand(g, rows, 1, 64, dtype=torch.bfloat16).to("cuda", torch.bfloat16) for _ in range(2))
    k.copy_(kk)
    v.copy_(vv)
    for nq in (1, 200):
        q = rand(g, nq, 2, 64, dtype=torch.bfloat16).to("cuda", torch.bfloat16)
        cu_q, cu_k = ends([nq]), ends([rows])
        assert torch.equal(sequence.packed_attention(q, k, v, cu_q, cu_k), sequence.packed_attention(q, kk, vv, cu_q, cu_k))
        far = [t.detach().requires_grad_(True) for t in (q, k, v)]
        near = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
        got, want = (torch.autograd.grad(sequence.packed_attention(*t, cu_q, cu_k), t, q) for t in (far, near))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del big


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    for kind in ("norm", "rope", "attention"):
        _, make = train_call(kind)
        args = make(1)
        leaf = args[0].detach().requires_grad_(True)
        out = {"norm": lambda: sequence.rms_norm(leaf, args[1]), "rope": lambda: sequence.rotary_axes(leaf, None, args[2], (16, 8, 8)),
               "attention": lambda: sequence.packed_attention(leaf, args[1], args[2], args[4], args[5])}[kind]()
        g = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="once_differentiable|differentiate"):
            torch.autograd.grad(g.float().sum(), leaf)


def two_streams(call, make):
    """The same call on two streams at once and on the default one: equal results."""
    a, b = make(1), make(2)
    want = [call(*a), call(*b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, (s, args) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(call(*args))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(g, want[i]))


def train_call(kind):
    if kind == "norm":
        def call(x, w, r, g):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, r)]
            y, h = sequence.rms_norm(leaves[0], leaves[1], residual=leaves[2])
            return (y, h) + torch.autograd.grad((y, h), leaves, (g, g))
        make = lambda s: (lambda g: [torch.randn(*d, generator=g).cuda() for d in ((300, 256), (256,), (300, 256), (300, 256))])(gen(s))      # noqa: E731
    elif kind == "rope":
        def call(q, k, pos, g):
            leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True)]
            out = sequence.rotary_axes(*leaves, pos, (16, 8, 8))
            return out + torch.autograd.grad(out, leaves, (g, g[:, :1].contiguous()))
        make = lambda s: (lambda g: [torch.randn(300, 2, 64, generator=g).cuda(), torch.randn(300, 1, 64, generator=g).cuda(),      # noqa: E731
                                     torch.randint(0, 5000, (3, 300), generator=g).cuda(), torch.randn(300, 2, 64, generator=g).cuda()])(gen(s))
    else:
        nq, nk, hk = (300, 300, 1) if kind == "attention" else (2, 3000, 2)

        def call(q, k, v, g, cu_q, cu_k):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = sequence.packed_attention(*leaves, cu_q, cu_k, max_q=nq, max_k=nk)
            return (out,) + torch.autograd.grad(out, leaves, g)
        make = lambda s: (lambda g: [torch.randn(2 * nq, 2, 64, generator=g).cuda().bfloat16(), torch.randn(2 * nk, hk, 64, generator=g).cuda().bfloat16(),      # noqa: E731
                                     torch.randn(2 * nk, hk, 64, generator=g).cuda().bfloat16(), torch.randn(2 * nq, 2, 64, generator=g).cuda().bfloat16(),
                                     ends([nq, nq]), ends([nk, nk])])(gen(s))
    return call, make


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["norm", "rope", "attention", "attention_few"])
def test_calls_on_two_streams_at_once(kind):
    two_streams(*train_call(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["norm", "rope", "attention", "attention_few"])
def test_captured_forward_and_backward_replay(kind):
    """Two graphs of the same call, replayed in turn with other inputs and eager work in between, against the eager call."""
    call, make = train_call(kind)
    inputs = [make(1), make(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for args in inputs:
            call(*args)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for args in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(*args))
        graphs.append(graph)
    for step in range(4):
        fresh = [make(10 + 2 * step + i) for i in range(2)]
        for old, new in zip(inputs, fresh):
            for a, b in zip(old, new):
                a.copy_(b)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, args in zip(outs, fresh):
            want = call(*args)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["norm", "rope", "attention"])
def test_gradients_against_differences(kind):
    """<gradient, d> against (f(x + e d) - f(x - e d)) / 2 e for a random direction d, in fp32 with sums in 64 bits.  The difference is off by
    e^2 / 6 times the third derivative along d and by the forward's fp32 error over e: with e = 2^-6 and derivatives of the order of
    f itself both stay below 1e-3 of the terms that are summed."""
    g = gen(21)
    if kind == "norm":
        x = [torch.randn(6, 64, generator=g).cuda(), torch.randn(64, generator=g).cuda(), torch.randn(6, 64, generator=g).cuda()]
        f = lambda x, w, r: sequence.rms_norm(x, w, residual=r)      # noqa: E731
    elif kind == "rope":
        x = [torch.randn(6, 2, 32, generator=g).cuda(), torch.randn(6, 1, 32, generator=g).cuda()]
        pos = torch.randint(0, 100, (2, 6), generator=g).cuda()
        f = lambda q, k: sequence.rotary_axes(q, k, pos, (6, 4), pairing="halves")      # noqa: E731
    else:
        x = [torch.randn(40, 4, 32, generator=g).cuda(), torch.randn(40, 2, 32, generator=g).cuda(), torch.randn(40, 2, 32, generator=g).cuda()]
        f = lambda q, k, v: (sequence.packed_attention(q, k, v, ends([25, 15])),)      # noqa: E731
    x = [t.requires_grad_(True) for t in x]
    outs = f(*x)
    weights = [torch.randn(o.shape, generator=g).cuda() for o in outs]
    grads = torch.autograd.grad(outs, x, weights)
    value = lambda ts: sum((o.double() * w.double()).sum().item() for o, w in zip(f(*ts), weights))      # noqa: E731
    e = 2.0 ** -6
    for i, t in enumerate(x):
        d = torch.randn(t.shape, generator=g).cuda()
        with torch.no_grad():
            up, down = ([u + s * e * d if j == i else u for j, u in enumerate(x)] for s in (1, -1))
            diff = (value(up) - value(down)) / (2 * e)
        terms = grads[i].double() * d.double()
        assert abs(terms.sum().item() - diff) <= 1e-3 * max(terms.abs().sum().item(), 1.0), (kind, i, terms.sum().item(), diff)


@pytest.mark.gpu
def test_a_block_of_the_operators_together():
    """norm -> fused projection with a LoRA adapter -> rotary positions -> attention -> projection, and back: the run of a pre-norm block, in
    fp32, against the same block in 64 bits on the CPU.  Every operator adds a few 2^-24 of its terms; through three projections of 128 terms
    each the bound of 2^-24 (3 * 128 + 1000) < 1e-4 of the largest result holds."""
    import lora_layers as L
    g = gen(31)
    width, hq, hk, d, lens = 128, 4, 2, 32, [37, 1, 60]
    T = sum(lens)
    x, r, gy = (torch.randn(T, width, generator=g) for _ in range(3))
    w = 1 + 0.1 * torch.randn(width, generator=g)
    wq, wo = torch.randn((hq + 2 * hk) * d, width, generator=g) / width ** 0.5, torch.randn(width, hq * d, generator=g) / width ** 0.5
    A, B = torch.randn(width, 4, generator=g) * 0.1, torch.randn(4, (hq + 2 * hk) * d, generator=g) * 0.1
    pos = torch.stack([torch.cat([torch.arange(n) for n in lens]) * s for s in (1, 3)]).int()

    lin = torch.nn.Linear(width, (hq + 2 * hk) * d, bias=False)
    lin.weight.data.copy_(wq)
    mod = L.LoRALinear(lin, rank=4, alpha=4)
    mod.lora.lora_A.data.copy_(A)
    mod.lora.lora_B.data.copy_(B)
    mod = mod.cuda()
    xs, rs, ws = (t.cuda().requires_grad_(True) for t in (x, r, w))
    cu = ends(lens)
    y, h = sequence.rms_norm(xs, ws, residual=rs)
    qkv = mod(y).view(T, hq + 2 * hk, d)
    q, k = sequence.rotary_axes(qkv[:, :hq], qkv[:, hq:hq + hk], pos.cuda(), (10, 6), pairing="halves")
    o = sequence.packed_attention(q, k, qkv[:, hq + hk:], cu, max_q=max(lens), max_k=max(lens))
    out = h + o.reshape(T, -1) @ wo.cuda().t()
    got = (out,) + torch.autograd.grad(out, (xs, rs, ws, mod.lora.lora_A, mod.lora.lora_B), gy.cuda())

    X, R, W, a, b = (t.double().requires_grad_(True) for t in (x, r, w, A, B))
    H = X + R
    Y = H * (H.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * W
    QKV = (Y @ wq.double().t() + Y @ a @ b).view(T, hq + 2 * hk, d)
    angle = pos.double()[[0] * 10 + [1] * 6].t() * torch.tensor([10000.0 ** (-i / 16) for i in range(16)], dtype=torch.float64)

    def turn(t):
        p, q = t[..., :16], t[..., 16:32]
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.cat([p * c - q * s, p * s + q * c, t[..., 32:]], -1)
    Q, K, V = turn(QKV[:, :hq]), turn(QKV[:, hq:hq + hk]), QKV[:, hq + hk:]
    outs, at = [], 0
    for n in lens:
        s = torch.einsum("ihd,jhd->hij", Q[at:at + n], K[at:at + n].repeat_interleave(2, 1)) * d ** -0.5
        p = s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf).softmax(-1)
        outs.append(torch.einsum("hij,jhd->ihd", p, V[at:at + n].repeat_interleave(2, 1)))
        at += n
    OUT = H + torch.cat(outs).reshape(T, -1) @ wo.double().t()
    want = (OUT,) + torch.autograd.grad(OUT, (X, R, W, a, b), gy.double())
    for name, t, u in zip(("out", "x", "r", "w", "A", "B"), got, want):
        assert (t.cpu().double() - u).abs().max() <= 1e-4 * u.abs().max(), name


# --------------------------------------------------------------------------------------------------- packed text tower
PROMPTS = ["crack", "a dog", "person", "cat"]


def tower(device, dtype, seed=0):
    from sam3_lora_amd.sam3_text import VETextEncoder
    lens = {p: n for p, n in zip(PROMPTS, (3, 9, 32, 1))}

    def tokenizer(texts, context_length):
        ids = torch.zeros(len(texts), context_length, dtype=torch.long)
        for row, t in enumerate(texts):
            n = lens[t]
            ids[row, :n] = torch.randint(1, 300, (n,), generator=gen(len(t)))
            if n > 4:
                ids[row, 2] = 0         # an id like the padding's in the middle of a prompt
        return ids
    torch.manual_seed(seed)
    enc = VETextEncoder(d_model=64, tokenizer=tokenizer, width=128, heads=4, layers=3, context_length=32, vocab_size=300, use_act_checkpoint=True)
    return enc.to(device, dtype)


def test_packed_text_switch_and_lengths_on_the_cpu():
    from sam3_lora_amd.sam3_text import VETextEncoder, set_packed_text
    ids = torch.tensor([[5, 6, 0, 7, 0, 0], [0, 0, 0, 0, 0, 0], [1, 2, 3, 4, 5, 6]])
    assert VETextEncoder._lengths(ids) == [4, 0, 6]
    enc = tower("cpu", torch.float32).eval()
    with torch.no_grad():
        want = enc(PROMPTS, device="cpu")
        assert set_packed_text(torch.nn.ModuleList([enc])) == 1 and enc.packed
        got = enc(PROMPTS, device="cpu")          # no GPU: the padded form
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("train", [False, True])
def test_packed_text_tower_equals_the_padded_one(train, dtype):
    """Three pre-norm blocks of 128: both forms round the same expressions at the same places in bf16 (2^-8 of values that the residual keeps
    near their start; a token passes 3 x 6 roundings) and differ in the order of fp32 sums otherwise (3 x 128 terms and more)."""
    from sam3_lora_amd.sam3_text import set_packed_text
    enc = tower("cuda", dtype)
    enc.train(train)
    g = torch.randn(32, len(PROMPTS), 64, generator=gen(3)).to("cuda", dtype)
    results = []
    for on in (False, True):
        set_packed_text(enc, on)
        enc.zero_grad()
        mask, memory, embeds = enc(PROMPTS, device="cuda")
        keep = ~mask.t()[..., None]
        if train:
            (memory * g * keep).float().sum().backward()
        results.append((mask, (memory * keep).detach(), embeds.detach(), {n: p.grad.clone() for n, p in enc.named_parameters() if p.grad is not None}))
    (m0, a, e0, g0), (m1, b, e1, g1) = results
    assert torch.equal(m0, m1) and torch.equal(e0, e1) and set(g0) == set(g1)
    tol = 18 * unit(dtype) if dtype == torch.bfloat16 else 2000 * F
    assert (a - b).float().abs().max() <= tol * a.float().abs().max()
    for n in g0:
        assert (g0[n] - g1[n]).float().norm() <= tol * max(g0[n].float().norm(), 1e-6), n


@pytest.mark.gpu
def test_packed_text_in_the_whole_model():
    """The tiny SAM3 image model in fp32: the loss does not change when its text tower runs packed (what the mask hides is not used)."""
    from sam3_lora_amd.sam3_data import SyntheticSegmentDataset, collate_fn_api
    from sam3_lora_amd.sam3_image import TINY_CONFIG, build_sam3_image_model
    from sam3_lora_amd.sam3_text import set_packed_text
    from sam3_lora_amd.trainer import build_criterion, match_all_steps, move_to_device
    cfg = dict(TINY_CONFIG, text=dict(TINY_CONFIG["text"], vocab_size=49408, context_length=32))
    ds = SyntheticSegmentDataset(2, resolution=112, source=128)
    batch = move_to_device(collate_fn_api([ds[0], ds[1]], dict_key="input", with_seg_masks=True)["input"], "cuda")
    model = build_sam3_image_model(device="cpu", eval_mode=False, config=cfg, match_in_forward=False, act_checkpoint=False, seed=6).to("cuda").train()
    _, wrapper = build_criterion("local")
    losses = []
    for on in (False, True):
        assert set_packed_text(model, on) == 1
        torch.manual_seed(0)
        out = model(batch)
        targets = [model.back_convert(t) for t in batch.find_targets]
        match_all_steps(wrapper, out.output, targets)
        losses.append(float(wrapper(out, targets)["core_loss"].detach()))
    assert abs(losses[0] - losses[1]) <= 1e-4 * abs(losses[0]), losses
