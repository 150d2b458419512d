"""
Sequence operators (sam3_lora_amd/sequence.py) at the edges of what their documentation allows: very many sequences, values that are not
finite, derivatives that do not exist.  Tolerances as in test_sequence.py.
"""
import math

import pytest
import torch

from sam3_lora_amd import _ffi, sequence
from test_sequence import DT, attn_ref, close, ends, gen, ids, rand, unit


# -------------------------------------------------------------------------------------------------- very many sequences
@pytest.mark.parametrize("tq,tk,b,hq,hk,max_q,max_k", [
    (64000, 64000, 4000, 16, 16, 64000, 64000), (262144, 262144, 512, 32, 8, 262144, 262144),        # nobody said how long they are
    (49000, 49000, 1101, 32, 8, 32768, 32768), (49000, 49000, 1101, 8, 1, 32768, 32768),              # one long one among short ones
    (130000, 130000, 65000, 16, 16, 130000, 130000), (65000, 1 << 22, 65000, 8, 8, 65000, 1 << 22), (1 << 22, 4096, 4096, 32, 8, 1 << 22, 4096),
    (41472, 41472, 8, 16, 16, 5184, 5184), (24, 400000, 24, 32, 8, 1, 32768), (24, 400000, 24, 32, 8, 24, 400000), (0, 0, 0, 2, 2, 0, 0), (5, 0, 1, 2, 1, 5, 0)])
def test_launches_are_as_large_as_the_rows_ask_for(tq, tk, b, hq, hk, max_q, max_k):
    """A launch has fewer than 2^32 threads (256 in a workgroup at most), and no more than a small multiple of the tiles that so many rows in so
    many sequences can have, whatever is said of the longest one."""
    lib = _ffi.load()
    for kernel, rows, heads in ((0, tq * (hq // hk), hk), (1, tq * (hq // hk), hk), (2, tk, hk)):
        n = lib.sam3_seq_attn_workgroups(kernel, tq, tk, b, hq, hk, 64, max_q, max_k, 0)
        most = heads * (rows // 128 + b)
        assert 0 < n < (1 << 32) // 256
        assert n <= 4 * most + 16384, (kernel, n, most)         # (chunks of keys: up to 8192 more)


def test_the_backwards_tiles_follow_the_type_and_the_head():
    """Eight pairs of 2048 (128 tiles of 128 rows or keys): tiles of 32, but for heads over 64 in fp32, where 128 are many enough."""
    f = _ffi.load().sam3_seq_attn_workgroups
    for d, dtype, wide in ((64, 0, False), (128, 0, False), (64, 1, False), (72, 1, True), (128, 1, True)):
        for kernel in (1, 2):
            assert f(kernel, 2048, 2048, 1, 8, 8, d, 2048, 2048, dtype) - f(kernel, 2048, 2048, 1, 8, 8, d, 0, 0, dtype) == 8 * ((16 if wide else 64) - 1)


def test_launches_that_do_not_exist_are_refused():
    import ctypes
    lib, p = _ffi.load(), ctypes.c_void_p(64)
    assert lib.sam3_seq_attn_workgroups(3, 8, 8, 1, 2, 2, 64, 8, 8, 0) == -22
    assert lib.sam3_seq_attn_workgroups(0, 8, 8, 1, 3, 2, 64, 8, 8, 0) == -22
    # 65000 sequences of 1024 key heads: 66.6 million workgroups
    for kernel in range(3):
        assert lib.sam3_seq_attn_workgroups(kernel, 130000, 130000, 65000, 1024, 1024, 8, 130000, 130000, 0) == -95
    assert lib.sam3_seq_attn_fwd(p, 8192, 8, p, 8192, 8, p, 8192, 8, p, p, None, p, None, None, 130000, 130000, 65000, 1024, 1024, 8, 130000, 130000, 1, 0.1, 0,
                                 None, 0, None) == -95
    assert lib.sam3_seq_attn_bwd(*([p, 8192, 8] * 4), p, p, p, p, p, p, p, 130000, 130000, 65000, 1024, 1024, 8, 130000, 130000, 1, 0.1, 0, p, 1 << 40, None) == -95


def test_chunks_of_keys_take_a_bounded_workspace():
    """The chunks' results have room for every row of q: with a hint that is too small, or room behind the sequences, no more than 2 GiB."""
    need = _ffi.load().sam3_seq_attn_fwd_workspace_bytes
    for tq, b, hq, hk, max_q, max_k in ((1 << 20, 1, 32, 8, 1, 1 << 20), (8192, 64, 32, 8, 1, 32768), (1 << 22, 1, 8, 8, 4, 1 << 30), (65536, 24, 32, 8, 1, 1 << 17)):
        for d in (8, 64, 128):
            assert need(tq, b, hq, hk, d, max_q, max_k, 0) <= 1 << 31, (tq, d)
    assert need(24, 24, 32, 8, 128, 1, 32768, 0) == 24 * 32 * 520 * 32        # (chunks of 1024 keys, as without the bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
def test_one_token_each_in_a_buffer_with_very_much_room(dtype):
    g = gen(6)
    lk = [3000, 1, 700]
    q = torch.zeros(200_000, 8, 64, device="cuda", dtype=dtype)
    q[:3] = rand(g, 3, 8, 64, dtype=dtype)
    k, v = (rand(g, sum(lk), 2, 64, dtype=dtype).to("cuda", dtype) for _ in range(2))
    cu_q, cu_k = ends([1] * 3), ends(lk)
    out = sequence.packed_attention(q, k, v, cu_q, cu_k, max_q=1, max_k=3000)
    ref = attn_ref(q[:3].cpu().double(), k.cpu().double(), v.cpu().double(), [1] * 3, lk, True, 0.125, unit(dtype))
    close(out[:3], ref["o"], ref["to"], "out")
    assert not out[3:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("lens,hq,hk,d,causal", [([3, 0, 20, 7, 1, 0, 33, 12] * 150, 4, 2, 32, True), ([5] * 600 + [700] + [2] * 600, 14, 2, 64, True),
                                                 ([9, 1, 0, 17] * 300 + [150], 2, 2, 128, False)])
def test_very_many_sequences_without_hints(lens, hq, hk, d, causal, dtype):
    """Without hints every one of them could be as long as all rows: the tiles are listed by the bounds then."""
    tq = sum(lens) + 14         # rows in front of the first and behind the last
    g = gen(d)
    q, go = rand(g, tq, hq, d, dtype=dtype, scale=1.5), rand(g, tq, hq, d, dtype=dtype)
    k, v = rand(g, tq, hk, d, dtype=dtype), rand(g, tq, hk, d, dtype=dtype)
    lib = _ffi.load()
    pairs, tiles = len(lens) * hk, tq * (hq // hk) // 128
    for kernel in range(3):
        assert lib.sam3_seq_attn_workgroups(kernel, tq, tq, len(lens), hq, hk, d, tq, tq, 0) < pairs * tiles / 4
    cu = ends(lens) + 5
    leaves = [t.to("cuda", dtype).requires_grad_(True) for t in (q, k, v)]
    out, lse = sequence.packed_attention(*leaves, cu, causal=causal, return_lse=True)
    grads = torch.autograd.grad(out, leaves, go.to("cuda", dtype))
    inside = slice(5, 5 + sum(lens))
    ref = attn_ref(q[inside], k[inside], v[inside], lens, lens, causal, d ** -0.5, unit(dtype), go[inside])
    close(out[inside], ref["o"], ref["to"], "out")
    for n, t in zip(("gq", "gk", "gv"), grads):
        close(t[inside], ref[n], ref["t" + n], n)
    for t in (out,) + grads:
        assert not t[:5].any() and not t[5 + sum(lens):].any()
    assert (lse[:5] == -math.inf).all() and (lse[5 + sum(lens):] == -math.inf).all()
    with torch.no_grad():           # the same tiles, told how long they are
        assert torch.equal(sequence.packed_attention(*leaves, cu, causal=causal, max_q=max(lens), max_k=max(lens)), out)


# ------------------------------------------------------------------------------------------------------ very many tokens
def test_rotary_axes_refuses_more_tokens_than_a_launch_can_have():
    import ctypes
    lib, p = _ffi.load(), ctypes.c_void_p(64)
    turns, axis = (ctypes.c_double * 4)(), (ctypes.c_ubyte * 4)()
    for t in (1 << 46, (1 << 62) + 1):
        assert lib.sam3_seq_rotary(p, 8, 8, None, 0, 0, p, None, p, 0, 1, 0, 1, turns, axis, 4, 0, 0, t, 1, 0, 8, 0, None) == -95
        assert "tokens" in lib.sam3_seq_last_error().decode()


@pytest.mark.gpu
def test_rotary_axes_of_more_tokens_than_2_to_27():
    """Eight tokens to a workgroup of 256 would be 2^32 threads and more, which no launch has."""
    t = (1 << 27) + 4099
    q = torch.randn(4099, 1, 8, generator=gen(1)).to("cuda", torch.bfloat16).repeat((t + 4098) // 4099, 1, 1)[:t]
    pos = torch.arange(4099, device="cuda", dtype=torch.int32).repeat((t + 4098) // 4099)[None, :t]
    out = sequence.rotary_axes(q, None, pos, (4,))
    want = sequence.rotary_axes(q[:4099], None, pos[:, :4099], (4,))
    whole = t // 4099 * 4099
    assert torch.equal(out[:whole].view(-1, 4099, 1, 8), want.expand(whole // 4099, 4099, 1, 8).view(-1, 4099, 1, 8)) and torch.equal(out[whole:], want[:t - whole])


# ----------------------------------------------------------------------------------------------- values that are not finite
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_one_token_sees_an_infinite_value(value, d, dtype):
    """One token over its keys, in one chunk and in several: the value's infinity is the result's, whichever block of keys it lies in, and no other
    element changes."""
    g = gen(d)
    lk, hq, hk = [70, 33, 200, 2100, 5000], 4, 2
    q = rand(g, len(lk), hq, d, dtype=dtype).to("cuda", dtype)
    k, v = (rand(g, sum(lk), hk, d, dtype=dtype).to("cuda", dtype) for _ in range(2))
    cu_q, cu_k = ends([1] * len(lk)), ends(lk)

    def call(v):
        return sequence.packed_attention(q, k, v, cu_q, cu_k, max_q=1, max_k=max(lk))
    good = call(v)
    begin = 0
    for i, n in enumerate(lk):
        for at in {0, n // 2, n - 1, n - n % 32 - 1}:
            bad = v.clone()
            bad[begin + at, 1, 5] = value
            bad[begin + at, 1, 8] = -value
            out = call(bad)
            got = out[i, hq // hk:]
            want = good.clone()
            want[i, hq // hk:, 5], want[i, hq // hk:, 8] = got[:, 5], got[:, 8]
            assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num()), (n, at)
            if math.isnan(value):
                assert got[:, 5].isnan().all() and got[:, 8].isnan().all(), (n, at)
            else:
                assert (got[:, 5] == value).all() and (got[:, 8] == -value).all(), (n, at)
        begin += n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("times", [1, 300])
@pytest.mark.parametrize("nk", [1, 70, 1500])
def test_a_row_whose_scores_are_all_minus_infinity_is_not_one_that_sees_no_key(nk, times, dtype):
    """softmax of nothing but -inf is 0 / 0, as it is in the formulas; a row without keys gives zeros.  With 300 sequences more the tiles of 128 run."""
    g = gen(nk)
    lq, lk = [3, 2] + [5] * (times - 1), [nk, 0] + [7] * (times - 1)
    q, go = (rand(g, sum(lq), 2, 64, dtype=dtype).to("cuda", dtype) for _ in range(2))
    k, v = (rand(g, sum(lk), 1, 64, dtype=dtype).to("cuda", dtype) for _ in range(2))
    k[:nk, 0, 7] = k[:nk, 0, 7].abs() + 1
    q[2, 1, 7] = -math.inf              # the last row of the first sequence sees all of its keys, in one of its heads
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = sequence.packed_attention(*leaves, ends(lq), ends(lk), max_q=max(lq), max_k=max(lk), return_lse=True)
    assert out[2, 1].isnan().all() and lse[2, 1] == -math.inf
    assert torch.isfinite(out[2, 0]).all() and not out[3:5].any() and torch.isfinite(out[5:]).all()
    assert not out[0].any() if nk == 1 else torch.isfinite(out[:2]).all()
    gq, gk, gv = torch.autograd.grad(out, leaves, go)
    assert gq[2, 1].isnan().all() and gk[:nk].isnan().all() and gv[:nk].isnan().all()
    assert torch.isfinite(gq[2, 0]).all() and not gq[3:5].any() and torch.isfinite(gq[5:]).all() and torch.isfinite(gk[nk:]).all() and torch.isfinite(gv[nk:]).all()


def ieee_ref(q, k, v, go, lq, lk, dtype):
    """out and the gradients by the formulas in 64 bits, row by row over the keys that it sees, as infinities and NaN come out of them; and what
    their finite elements may be off by.  A score is a sum of d products (fp32), so a weight is off by 2 E of itself with E = (d + 8) F times
    the largest sum of |q k|, and once more by its rounding, u; dS = p (go v - D) by those, by D's (the rounded out, u, and the weights') and by a
    rounding of its own; the results by theirs, and by F for each row or key that is summed: 5 u + 5 E and less of the sum of absolute terms."""
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    c = d ** -0.5
    zero = lambda t: torch.zeros_like(t)      # noqa: E731
    got, size = [zero(t) for t in (q, q, k, v)], [zero(t) for t in (q, q, k, v)]
    fin = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs()      # noqa: E731
    a = b = 0
    most = 0.0
    for m, n in zip(lq, lk):
        for i in range(m):
            seen = min(max(i + 1 + n - m, 0), n)
            if seen == 0:
                continue
            for h in range(hq):
                kh = h // (hq // hk)
                K, V, Q, G = k[b:b + seen, kh], v[b:b + seen, kh], q[a + i, h], go[a + i, h]
                s = (K * Q).sum(1) * c
                most = max(most, ((fin(K) * fin(Q)).sum(1) * c).max().item())
                e = (s - s.max()).exp()
                p = e / e.sum()
                o = (p[:, None] * V).sum(0)
                ds = p * ((V * G).sum(1) - (G * o).sum())
                P = fin(p)
                O = (P[:, None] * fin(V)).sum(0)
                S = P * ((fin(V) * fin(G)).sum(1) + (fin(G) * O).sum())
                for t, (ro, rq, rk, rv) in ((got, (o, (ds[:, None] * K).sum(0) * c, ds[:, None] * Q * c, p[:, None] * G)),
                                            (size, (O, (S[:, None] * fin(K)).sum(0) * c, S[:, None] * fin(Q) * c, P[:, None] * fin(G)))):
                    t[0][a + i, h], t[1][a + i, h] = ro, rq
                    t[2][b:b + seen, kh] += rk
                    t[3][b:b + seen, kh] += rv
        a, b = a + m, b + n
    E = (d + 8 + max(lq) * (hq // hk) + max(lk)) * 2.0 ** -24 * (1 + most)
    return got, [(5 * unit(dtype) + 5 * E) * t for t in size]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("lq,lk,hq,hk,d,more", [([9], [9], 2, 1, 64, 0), ([40], [40], 2, 2, 32, 0), ([50], [90], 2, 1, 128, 0), ([3, 1], [140, 70], 4, 2, 64, 0),
                                                ([150], [150], 2, 2, 64, 0), ([150], [200], 1, 1, 128, 300), ([140], [140], 3, 1, 32, 300)])
@pytest.mark.parametrize("which", ["q", "k", "v", "go"])
def test_what_is_not_finite_reaches_what_the_formulas_say(which, lq, lk, hq, hk, d, more, dtype):
    """One infinity in a query, key, value or gradient: each element of the results is finite where the formulas' is, and right there; the others
    are infinite or NaN as theirs are, wherever the borders of blocks lie (a value's infinity and gv's keep their sign; D, the sum of infinities
    in another order, decides between the two in gq and gk)."""
    g = gen(d)
    tq, tk = sum(lq), sum(lk)
    q, go = rand(g, tq + 20 * more, hq, d, dtype=dtype), rand(g, tq + 20 * more, hq, d, dtype=dtype)
    k, v = rand(g, tk + 20 * more, hk, d, dtype=dtype), rand(g, tk + 20 * more, hk, d, dtype=dtype)
    q[:tq, :, 5] = q[:tq, :, 5].abs() + 0.125           # an infinite k is +-inf in all scores
    cu_q, cu_k = ends(lq + [20] * more), ends(lk + [20] * more)
    for at in {0, 1, lk[0] // 2, lk[0] - 1}:
        for value in (math.inf, -math.inf):
            t = dict(q=q.clone(), k=k.clone(), v=v.clone(), go=go.clone())
            row = min(at, lq[0] - 1) if which in ("q", "go") else at
            t[which][row, 0, 5] = value
            want, tol = ieee_ref(t["q"][:tq], t["k"][:tk], t["v"][:tk], t["go"][:tq], lq, lk, dtype)
            leaves = [t[n].to("cuda", dtype).requires_grad_(True) for n in ("q", "k", "v")]
            out = sequence.packed_attention(*leaves, cu_q, cu_k, max_q=max(lq + [20]), max_k=max(lk + [20]))
            got = (out,) + torch.autograd.grad(out, leaves, t["go"].to("cuda", dtype))
            for name, x, y, most in zip(("out", "gq", "gk", "gv"), got, want, tol):
                x, what = x.detach().cpu().double(), (which, at, value, name)
                assert torch.isfinite(x[len(y):]).all(), what
                x, fin = x[:len(y)], torch.isfinite(y)
                assert torch.equal(torch.isfinite(x), fin), what
                if name in ("out", "gv"):
                    assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x[~fin].nan_to_num(), y[~fin].nan_to_num()), what
                off = (x - y)[fin].abs() - most[fin]
                assert (off <= 0).all(), (what, off.max().item())


# ------------------------------------------------------------------------------------------- derivatives that do not exist
def operator_calls():
    g = gen(4)
    x, w = torch.randn(12, 64, generator=g).cuda(), torch.randn(64, generator=g).cuda()
    q, k, v = (torch.randn(12, 2, 32, generator=g).cuda() for _ in range(3))
    pos, cu = torch.arange(12, device="cuda", dtype=torch.float32)[None], ends([5, 7])
    return {"norm": (lambda *t: sequence.rms_norm(t[0], t[1], residual=t[2]), (x, w, x * 2)), "norm alone": (sequence.rms_norm, (x, w)),
            "rotary": (lambda *t: sequence.rotary_axes(t[0], t[1], t[2], (16,)), (q, k, pos)),
            "attention": (lambda *t: sequence.packed_attention(*t, cu), (q, k, v)),
            "lse": (lambda *t: sequence.packed_attention(*t, cu, return_lse=True), (q, k, v))}


@pytest.mark.gpu
def test_forward_derivatives_are_refused():
    """A dual tensor does not require a gradient; without its tangent the result would count as constant."""
    from torch.autograd import forward_ad
    for name, (call, args) in operator_calls().items():
        plain = call(*args)
        with forward_ad.dual_level():
            same = call(*args)              # nothing is dual
            assert all(torch.equal(a, b) for a, b in zip(*((t,) if torch.is_tensor(t) else t for t in (plain, same)))), name
            for i, t in enumerate(args):
                dual = list(args)
                dual[i] = forward_ad.make_dual(t, torch.ones_like(t))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises((NotImplementedError, RuntimeError)):
                        call(*dual)
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="gradient"):
        sequence.rms_norm_q8(forward_ad.make_dual(x, x), w)


@pytest.mark.gpu
def test_traced_calls_are_calls():
    """A trace holds the call, not the result of its example inputs."""
    for name, (call, args) in operator_calls().items():
        with torch.no_grad():
            traced = torch.jit.trace(call, args, check_trace=False)
        other = [t.flip(0) * 1.25 for t in args]
        got, want = traced(*other), call(*other)
        for a, b in zip(*((t,) if torch.is_tensor(t) else t for t in (got, want))):
            assert torch.equal(a, b), name
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with torch.no_grad(), pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda x: sequence.rms_norm_q8(x, w)[1], (x,), check_trace=False)


# --------------------------------------------------------------------------------------------------- packed text tower
def test_the_packed_tower_steps_back_where_it_would_miss_something():
    """Hooks of the modules that the packed form goes round, another forward, or another module in an attention's place."""
    import torch.nn as nn
    from test_sequence import tower
    enc = tower("cpu", torch.float32).encoder
    assert enc.packs()
    blk = enc.transformer.resblocks[1]
    for m in (enc, enc.transformer, blk, blk.attn):
        for register in (m.register_forward_hook, m.register_forward_pre_hook, m.register_full_backward_hook, m.register_full_backward_pre_hook):
            handle = register(lambda *a: None)
            assert not enc.packs()
            handle.remove()
            assert enc.packs()
        m.forward = m.forward
        assert not enc.packs()
        del m.forward
        assert enc.packs()
    for register in (nn.modules.module.register_module_forward_hook, nn.modules.module.register_module_full_backward_hook):
        handle = register(lambda *a: None)
        assert not enc.packs()
        handle.remove()
        assert enc.packs()
    blk.ln_1.register_forward_hook(lambda *a: None)         # these are called either way
    blk.mlp.c_fc.register_forward_hook(lambda *a: None)
    assert enc.packs()
    stock = blk.attn
    blk.attn = nn.MultiheadAttention(128, 4, batch_first=True)
    assert not enc.packs()
    blk.attn = nn.Identity()
    assert not enc.packs()
    blk.attn = stock
    assert enc.packs()


@pytest.mark.gpu
def test_hooks_see_the_tower_with_the_packed_switch_on():
    from sam3_lora_amd.sam3_text import set_packed_text
    from test_sequence import PROMPTS, tower
    enc = tower("cuda", torch.float32).eval()
    seen = []
    enc.encoder.transformer.resblocks[2].attn.register_forward_hook(lambda m, args, out: seen.append(out[0].shape))
    with torch.no_grad():
        want = enc(PROMPTS, device="cuda")
        set_packed_text(enc)
        got = enc(PROMPTS, device="cuda")
    assert len(seen) == 2 and seen[0] == seen[1] and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ the 8-bit image multiplied
@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,out,bias", [(1, 128, 64, True), (37, 1024, 256, True), (300, 512, 4096, False)])
def test_the_frozen_linear_takes_the_norms_image(rows, width, out, bias):
    """image x scales times the frozen weight's own image: products of 8-bit numbers are exact in fp32, their sum is off by (width + 1) F of the
    absolute terms, the scales and the bias by a few F, the result by one rounding to bf16."""
    from sam3_lora_amd import fp8
    g = gen(width)
    x, r = (rand(g, rows, width, dtype=torch.bfloat16, scale=s).to("cuda", torch.bfloat16) for s in (1, 3))
    weight = (rand(g, width, dtype=torch.bfloat16, scale=0.2) + 1).to("cuda", torch.bfloat16)
    w = rand(g, out, width, dtype=torch.bfloat16, scale=width ** -0.5).to("cuda", torch.bfloat16)
    b = rand(g, out, dtype=torch.bfloat16).to("cuda", torch.bfloat16) if bias else None
    with torch.no_grad():
        image, scales, h = sequence.rms_norm_q8(x, weight, residual=r)
        y = fp8.fp8_linear_q(image, scales, w, b)
    st = fp8.state_for(w)
    a, c = image.float().double() * scales.double(), st.wq.float().double() * st.scale.double()
    want = a @ c.t() + (0 if b is None else b.double())
    terms = a.abs() @ c.t().abs() + (0 if b is None else b.double().abs())
    close(y, want.cpu(), (unit(torch.bfloat16) * want.abs() + (width + 8) * 2.0 ** -24 * terms).cpu(), "y")


# ------------------------------------------------------------------------------------------------------- far positions
@pytest.mark.gpu
def test_angles_of_far_positions_against_fifty_digits():
    """Up to 2^30 an angle is off by 2^-24 of a turn, and by the fp32 functions (a rounding of half a turn's fraction, 2 ulp) behind that; at 2^40
    by 2^-14 of a turn."""
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    positions = [0, 1, -5, 12345, (1 << 20) + 7, (1 << 30) - 1, -(1 << 30) + 3, (1 << 29) + 12345, (1 << 40) - 9, 10 ** 12]
    pairs = 16
    q = torch.zeros(len(positions), 1, 2 * pairs, device="cuda")
    q[..., 0::2] = 1.0
    got = sequence.rotary_axes(q, None, torch.tensor([positions], device="cuda"), (pairs,))[:, 0].cpu().double()
    for t, pos in enumerate(positions):
        for i in range(pairs):
            turns = Decimal(pos) * (Decimal(10000).ln() * Decimal(-i) / Decimal(pairs)).exp() / (2 * pi)
            angle = 2 * math.pi * float(turns - turns.to_integral_value())
            tol = 2 * math.pi * 2.0 ** -24 * max(1.0, abs(pos) / 2.0 ** 30) + (math.pi / 2 + 4) * 2.0 ** -24
            assert abs(got[t, 2 * i].item() - math.cos(angle)) <= tol and abs(got[t, 2 * i + 1].item() - math.sin(angle)) <= tol, (pos, i)


# ------------------------------------------------------------------------------------------------ sizes as programs have them
@pytest.mark.gpu
def test_lengths_and_sections_of_other_integer_types():
    """Lengths as numpy's reductions give them are lengths; sections that are not whole numbers are refused, not cut off."""
    import numpy as np
    g = gen(8)
    lens = np.array([5, 40, 9])
    q, k, v = (torch.randn(54, 2, 32, generator=g).cuda() for _ in range(3))
    cu = ends(lens.tolist())
    want = sequence.packed_attention(q, k, v, cu, max_q=40, max_k=40)
    for m in (lens.max(), np.int32(40), np.uint16(40)):
        assert torch.equal(sequence.packed_attention(q, k, v, cu, max_q=m, max_k=m), want)
    for m in (40.0, np.float32(40), -np.int64(1), torch.tensor(40), "40"):
        with pytest.raises(ValueError, match="length"):
            sequence.packed_attention(q, k, v, cu, max_q=m)
    pos = torch.arange(54, device="cuda")[None].expand(2, 54)
    turned = sequence.rotary_axes(q, None, pos, (8, 4))
    assert torch.equal(sequence.rotary_axes(q, None, pos, np.array([8, 4])), turned) and torch.equal(sequence.rotary_axes(q, None, pos, [8, 4]), turned)
    for sections in ([8.7, 4], (8.7, 4), [torch.tensor(8.0), 4]):
        with pytest.raises(TypeError):
            sequence.rotary_axes(q, None, pos, sections)


# ------------------------------------------------------------------------------------------------------ captured calls
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["many", "few"])
def test_a_captured_call_follows_the_bounds_of_each_replay(kind):
    """Without hints (tiles listed by the bounds), and one token each over chunks of keys: the lengths lie on the GPU, and a replay takes those that
    lie there then; two graphs of the same call in turn with eager work between."""
    g = gen(9)
    rng = torch.Generator().manual_seed(5)
    b, tq, tk, hq, hk = (700, 3000, 3000, 2, 1) if kind == "many" else (3, 3, 9000, 4, 2)
    q, go = (torch.randn(tq, hq, 64, generator=g).cuda().bfloat16() for _ in range(2))
    k, v = (torch.randn(tk, hk, 64, generator=g).cuda().bfloat16() for _ in range(2))
    how = {} if kind == "many" else dict(max_q=1, max_k=4000)

    def bounds(total):
        cut = torch.randint(0, total + 1, (b - 1,), generator=rng).sort().values
        return torch.cat([torch.zeros(1, dtype=torch.long), cut, torch.tensor([total])]).int().cuda()

    def call(q, k, v, cu_q, cu_k):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out, lse = sequence.packed_attention(*leaves, cu_q, cu_k, return_lse=True, **how)
        return (out, lse) + torch.autograd.grad(out, leaves, go)
    inputs = []
    for _ in range(2):
        cu = bounds(tq) if kind == "many" else ends([1] * 3)
        inputs.append([q.clone(), k.clone(), v.clone(), cu, cu.clone() if kind == "many" else bounds(tk)])
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
    for _ in range(4):
        for args in inputs:
            args[0].copy_(args[0].flip(0))
            cu = bounds(tk)
            args[4].copy_(cu)
            if kind == "many":
                args[3].copy_(cu)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, args in zip(outs, inputs):
            assert all(torch.equal(a, c) for a, c in zip(out, call(*args)))


# ------------------------------------------------------------------------------------------------------- partial gradients
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("times", [1, 150])
def test_attention_gradients_one_by_one(times, dtype):
    """Each gradient alone has the bits that it has among the others; frozen keys and values cost neither their kernel nor its tensors."""
    g = gen(15)
    lens = [90, 33, 0, 7] * times
    q, go = (rand(g, sum(lens), 4, 64, dtype=dtype).to("cuda", dtype) for _ in range(2))
    k, v = (rand(g, sum(lens), 2, 64, dtype=dtype).to("cuda", dtype) for _ in range(2))
    cu = ends(lens)

    def grads(*need):
        leaves = [t.detach().requires_grad_(n) for t, n in zip((q, k, v), need)]
        out = sequence.packed_attention(*leaves, cu, max_q=90, max_k=90)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(out, [t for t, n in zip(leaves, need) if n], go)
        return got, torch.cuda.max_memory_allocated() - before
    (gq, gk, gv), most = grads(True, True, True)
    for need, want in (((True, False, False), (gq,)), ((False, True, False), (gk,)), ((False, False, True), (gv,)), ((True, False, True), (gq, gv)), ((False, True, True), (gk, gv))):
        got, peak = grads(*need)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if need == (True, False, False):
            assert peak <= most - 2 * k.numel() * k.element_size() + 4096


def test_gradients_of_keys_without_those_of_values_are_refused():
    import ctypes
    lib, p = _ffi.load(), ctypes.c_void_p(64)
    for gk, gv in ((None, p), (p, None)):
        assert lib.sam3_seq_attn_bwd(*([p, 64, 64] * 4), p, p, p, p, p, gk, gv, 8, 8, 1, 4, 4, 64, 8, 8, 1, 0.1, 0, p, 1 << 20, None) == -22


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT, ids=ids)
@pytest.mark.parametrize("bad", ["q", "k", "v", "go", "all"])
def test_nothing_but_nan_comes_out_as_nan(bad, dtype):
    """A step that has diverged: whole tensors of NaN, at sizes where every block of the border holds some."""
    g = gen(17)
    lens = [700, 33, 260] * 20
    t = {n: rand(g, sum(lens), h, 64, dtype=dtype).to("cuda", dtype) for n, h in (("q", 4), ("k", 2), ("v", 2), ("go", 4))}
    for n in t:
        if bad in (n, "all"):
            t[n].fill_(math.nan)
    cu = ends(lens)
    leaves = [t[n].requires_grad_(True) for n in ("q", "k", "v")]
    out = sequence.packed_attention(*leaves, cu, max_q=700, max_k=700)
    gq, gk, gv = torch.autograd.grad(out, leaves, t["go"])
    assert out.isnan().all() if bad != "go" else torch.isfinite(out).all()
    assert gq.isnan().all() and gk.isnan().all()
    assert gv.isnan().all() if bad != "v" else torch.isfinite(gv).all()
