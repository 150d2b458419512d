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
        n = lib.sam3_seq_attn_workgroups(kernel, tq, tk, b, hq, hk, max_q, max_k)
        most = heads * (rows // 128 + b)
        assert 0 < n < (1 << 32) // 256
        assert n <= 4 * most + 16384, (kernel, n, most)         # (chunks of keys: up to 8192 more)


def test_launches_that_do_not_exist_are_refused():
    import ctypes
    lib, p = _ffi.load(), ctypes.c_void_p(64)
    assert lib.sam3_seq_attn_workgroups(3, 8, 8, 1, 2, 2, 8, 8) == -22
    assert lib.sam3_seq_attn_workgroups(0, 8, 8, 1, 3, 2, 8, 8) == -22
    # 65000 sequences of 1024 key heads: 66.6 million workgroups
    for kernel in range(3):
        assert lib.sam3_seq_attn_workgroups(kernel, 130000, 130000, 65000, 1024, 1024, 130000, 130000) == -95
    assert lib.sam3_seq_attn_fwd(p, 8192, 8, p, 8192, 8, p, 8192, 8, p, p, None, p, None, None, 130000, 130000, 65000, 1024, 1024, 8, 130000, 130000, 1, 0.1, 0,
                                 None, 0, None) == -95
    assert lib.sam3_seq_attn_bwd(*([p, 8192, 8] * 4), p, p, p, p, p, p, p, 130000, 130000, 65000, 1024, 1024, 8, 130000, 130000, 1, 0.1, 0, p, 1 << 40, None) == -95


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
        assert lib.sam3_seq_attn_workgroups(kernel, tq, tq, len(lens), hq, hk, tq, tq) < pairs * tiles / 4
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
