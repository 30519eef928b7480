"""Rotary positions: frequencies and refusals on the CPU, the kernel against the formula in 64 bits on the GPU."""
import ctypes as C
import math

import numpy as np
import pytest

SCALINGS = {
    "none": {},
    "linear": dict(factor=4.0),
    "base": dict(factor=8.0),
    "bands": dict(factor=8.0, original_context=8192, low_freq_factor=1.0, high_freq_factor=4.0),
    "ramp": dict(factor=16.0, original_context=4096, beta_fast=32.0, beta_slow=1.0),
}


def expected_frequencies(rot, theta, scaling, **kw):
    """The formulas of include/drkv.h, pair by pair, and the factor a.  In 80 bits: at position 2^31 a double's frequency
    would be off by some 10^-6 rad."""
    L = np.longdouble
    factor, theta, pi = L(kw.get("factor", 1.0)), L(theta), L("3.14159265358979323846264338327950288")
    base = theta * factor ** (L(rot) / (rot - 2)) if scaling == "base" else theta
    out = []
    if scaling == "ramp":
        pair_of = lambda turns: rot * np.log(kw["original_context"] / (turns * 2 * pi)) / (2 * np.log(theta))
        low, high = max(np.floor(pair_of(kw["beta_fast"])), 0), min(np.ceil(pair_of(kw["beta_slow"])), rot - 1)
    for i in range(rot // 2):
        f = base ** (-2 * L(i) / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "bands":
            n = kw["original_context"] * f / (2 * pi)
            lo, hi = kw["low_freq_factor"], kw["high_freq_factor"]
            if n <= lo:
                f /= factor
            elif n < hi:
                keep = (n - lo) / (hi - lo)
                f = f * keep + f / factor * (1 - keep)
        if scaling == "ramp":
            r = min(max((i - low) / max(high - low, L(0.001)), L(0)), L(1))
            f = f / factor * r + f * (1 - r)
        out.append(f)
    return np.array(out), 0.1 * math.log(float(factor)) + 1.0 if scaling == "ramp" else 1.0


def rotate64(x, pos, freq, a, layout, inverse):
    """x [tokens, heads, d] in float64; returns the rotated rows and |x0| + |x1| spread over both members of a pair."""
    rot = 2 * len(freq)
    angle = pos.astype(np.longdouble)[:, None] * freq[None, :]
    c, s = a * np.cos(angle).astype(np.float64)[:, None, :], a * np.sin(angle).astype(np.float64)[:, None, :] * (-1 if inverse else 1)
    y, mag = x.copy(), np.zeros_like(x)
    i0, i1 = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "halves" else (slice(0, rot, 2), slice(1, rot, 2))
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    mag[..., i0] = mag[..., i1] = np.abs(x0) + np.abs(x1)
    return y, mag


@pytest.mark.parametrize("scaling", sorted(SCALINGS))
@pytest.mark.parametrize("rot", [8, 50, 64, 128])
def test_frequencies(drkv_lib, scaling, rot):
    from deusridet_b200 import Rope
    want, _ = expected_frequencies(rot, 5e5, scaling, **SCALINGS[scaling])
    got = Rope(head_dim=128, rotary_dim=rot, theta=5e5, scaling=scaling, device=-1, **SCALINGS[scaling]).frequencies()
    # both in 80 bits, one rounding to double
    np.testing.assert_allclose(got, want.astype(np.float64), rtol=2.0 ** -52, atol=0)


def test_refusals(drkv_lib):
    from deusridet_b200 import DrkvError, Rope, capi
    for bad in (dict(head_dim=12), dict(head_dim=520), dict(head_dim=0), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=7),
                dict(head_dim=64, rotary_dim=0), dict(head_dim=64, theta=1.0), dict(head_dim=64, theta=float("nan")),
                dict(head_dim=64, scaling="linear", factor=0.5), dict(head_dim=64, scaling="linear", factor=float("inf")),
                dict(head_dim=64, rotary_dim=2, scaling="base", factor=2.0), dict(head_dim=64, scaling="bands", factor=2.0),
                dict(head_dim=64, scaling="bands", factor=2.0, original_context=8192, low_freq_factor=4.0, high_freq_factor=4.0),
                dict(head_dim=64, scaling="ramp", factor=2.0, original_context=8192, beta_fast=1.0, beta_slow=2.0),
                dict(head_dim=64, attention_factor=-1.0)):
        with pytest.raises(DrkvError) as err:
            Rope(device=-1, **bad)
        assert err.value.code == capi.ERR_INVALID, bad
    for bad in (dict(layout="thirds"), dict(scaling="cubic"), dict(dtype="f32")):
        with pytest.raises(ValueError):
            Rope(head_dim=64, device=-1, **bad)
    rope = Rope(head_dim=64, device=-1)
    rows = capi.RopeRows(4096, 8192, 1, 64, 64, 64, 64)
    assert drkv_lib.drkv_rope_apply(rope.h, 1, 4096, C.byref(rows), None, 0, None) == capi.ERR_NO_DEVICE
    assert drkv_lib.drkv_rope_apply(None, 1, 4096, C.byref(rows), None, 0, None) == capi.ERR_INVALID
    assert drkv_lib.drkv_rope_apply(rope.h, -1, 4096, C.byref(rows), None, 0, None) == capi.ERR_INVALID
    assert drkv_lib.drkv_rope_apply(rope.h, 1, 4096, None, None, 0, None) == capi.ERR_INVALID
    rope.close()
    rope.close()


def _check(got, x, pos, freq, a, layout, inverse, dtype):
    import torch
    want, mag = rotate64(x.double().cpu().numpy(), pos.cpu().numpy(), freq, a, layout, inverse)
    half_step = torch.finfo(dtype).eps / 2
    # one rounding of the result (and of subnormal fp16 results, 2^-25), plus fp32 work: cosine and sine within 2 units
    # of 2^-24 and the phase's 2^-25 half turns, two products and a sum
    tol = np.abs(want) * half_step + 2.0 ** -25 + 1e-6 * a * mag
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol * (1 + 1e-3)).all(), float((err - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("d,rot", [(128, 128), (256, 64), (64, 50), (64, 26), (80, 72), (8, 2), (512, 512), (128, 8)])
@pytest.mark.parametrize("tokens,inverse", [(1, False), (7, True), (300, False)])
def test_against_formula(drkv_lib, dtype, layout, d, rot, tokens, inverse):
    import torch
    from deusridet_b200 import Rope
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator(device="cuda").manual_seed(d * 1000 + rot + tokens)
    scaling = sorted(SCALINGS)[(d + rot + tokens) % 5] if rot >= 8 else "linear"
    rope = Rope(head_dim=d, rotary_dim=rot, theta=1e6, layout=layout, dtype=dtype, scaling=scaling, device=0, **SCALINGS[scaling])
    freq, a = expected_frequencies(rot, 1e6, scaling, **SCALINGS[scaling])
    hq, hkv = 6, 2
    fused = torch.randn(tokens, (hq + 2 * hkv) * d, generator=g, device="cuda").to(t)
    q, k = fused[:, :hq * d].unflatten(1, (hq, d)), fused[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    # far positions, the largest one, the first ones and a negative one
    pos = torch.randint(-5, 2 ** 31 - 1, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = 2 ** 31 - 1 if tokens > 1 else 1000003
    before = fused.clone()
    q_out, k_out = rope.apply(pos, q, k, inverse=inverse)
    torch.cuda.synchronize()
    assert torch.equal(fused, before)
    _check(q_out, q, pos, freq, a, layout, inverse, t)
    _check(k_out, k, pos, freq, a, layout, inverse, t)
    assert torch.equal(q_out[..., rot:], q[..., rot:])
    # in place on the strided rows: the same bits, and the rows that are not rotated stay
    rope.apply(pos, q, k, out_q=q, out_k=k, inverse=inverse)
    torch.cuda.synchronize()
    assert torch.equal(q, q_out) and torch.equal(k, k_out)
    assert torch.equal(fused[:, (hq + hkv) * d:], before[:, (hq + hkv) * d:])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("d,rot,hq,hkv,tokens", [(128, 128, 64, 8, 1), (128, 34, 60, 5, 5), (64, 62, 33, 0, 2), (256, 142, 19, 4, 40),
                                                 (128, 116, 31, 1, 2500), (64, 2, 3, 3, 700), (96, 90, 50, 7, 3)])
def test_many_heads_few_tokens_odd_halves(drkv_lib, layout, d, rot, hq, hkv, tokens):
    """Heads spread over several CTAs (the last with fewer), halves that begin inside a 16-byte vector; out of place and in place."""
    import torch
    from deusridet_b200 import Rope
    g = torch.Generator(device="cuda").manual_seed(d + rot + tokens)
    rope = Rope(head_dim=d, rotary_dim=rot, theta=1e4, layout=layout, dtype="f16", device=0)
    freq, a = expected_frequencies(rot, 1e4, "none")
    q = torch.randn(tokens, hq, d, generator=g, device="cuda").half()
    k = torch.randn(tokens, hkv, d, generator=g, device="cuda").half() if hkv else None
    pos = torch.randint(0, 2 ** 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    q_out, k_out = rope.apply(pos, q, k)
    _check(q_out, q, pos, freq, a, layout, False, torch.float16)
    assert torch.equal(q_out[..., rot:], q[..., rot:])
    if hkv:
        _check(k_out, k, pos, freq, a, layout, False, torch.float16)
    keep = torch.nan * torch.ones(tokens, hq + 1, d, device="cuda", dtype=torch.float16)      # a head behind, left as it was
    keep[:, :hq] = q
    rope.apply(pos, keep[:, :hq], k, out_q=keep[:, :hq], out_k=k)
    torch.cuda.synchronize()
    assert torch.equal(keep[:, :hq], q_out) and torch.isnan(keep[:, hq]).all()
    assert k is None or torch.equal(k, k_out)


@pytest.mark.gpu
def test_strides_orders_alignment(drkv_lib):
    """Head-major storage, rows starting at odd elements, one tensor only, k alone, no tokens."""
    import torch
    from deusridet_b200 import Rope
    rope = Rope(head_dim=64, dtype="f16", device=0)
    freq, a = expected_frequencies(64, 1e4, "none")
    g = torch.Generator(device="cuda").manual_seed(3)
    pos = torch.arange(100, 133, device="cuda", dtype=torch.int32)
    head_major = torch.randn(5, 33, 64, generator=g, device="cuda").half().transpose(0, 1)
    out, none = rope.apply(pos, head_major, out_q=torch.empty_like(head_major))
    assert none is None
    _check(out, head_major, pos, freq, a, "halves", False, torch.float16)
    for shift in (1, 2, 4):
        base = torch.randn(33, 2 * 67, generator=g, device="cuda").half()
        odd = base[:, shift:shift + 128].unflatten(1, (2, 64))
        _, out = rope.apply(pos, None, odd)
        _check(out, odd, pos, freq, a, "halves", False, torch.float16)
    expanded = torch.randn(33, 1, 64, generator=g, device="cuda").half().expand(33, 4, 64)     # one row for four heads
    out, _ = rope.apply(pos, expanded)
    _check(out, expanded, pos, freq, a, "halves", False, torch.float16)
    empty = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    rope.apply(pos[:0], empty)
    no_heads = torch.empty(33, 0, 64, device="cuda", dtype=torch.float16)
    rope.apply(pos, no_heads, expanded)


@pytest.mark.gpu
def test_streams(drkv_lib):
    """The current stream by default (a capture too), a given one as an object or a handle, with outputs allocated for it."""
    import torch
    from deusridet_b200 import Rope
    rope = Rope(head_dim=128, dtype="bf16", device=0)
    pos = torch.arange(4000, device="cuda", dtype=torch.int32)
    q = torch.randn(4000, 8, 128, device="cuda").bfloat16()
    want, _ = rope.apply(pos, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            x = q + 0
            got, _ = rope.apply(pos, x, out_q=x)                     # in place right behind the copy, on its stream
    side.synchronize()
    assert torch.equal(got, want)
    for stream in (side, side.cuda_stream, torch.cuda.default_stream().cuda_stream):
        torch.cuda.synchronize()
        got, _ = rope.apply(pos, q, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = rope.apply(pos, q)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_argument_checks_on_tensors(drkv_lib):
    import torch
    from deusridet_b200 import DrkvError, Rope
    rope = Rope(head_dim=64, dtype="bf16", device=0)
    pos = torch.arange(4, device="cuda", dtype=torch.int32)
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (dict(q=x.half()), dict(q=x.cpu()), dict(q=x[:3]), dict(q=x[..., :32]), dict(q=x, out_q=x[:, :1]),
                dict(q=None), dict(k=x, out_q=x), dict(q=x.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            rope.apply(pos, **bad)
    with pytest.raises(ValueError):
        rope.apply(pos.long(), x)
    with pytest.raises(ValueError):
        rope.apply(pos.cpu(), x)
    buf = torch.zeros(16, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(DrkvError):                                       # in place with other strides
        rope.apply(pos, buf[:4], out_q=buf[0:8:2])
    with pytest.raises(DrkvError):                                       # overlapping by a row
        rope.apply(pos, buf[:4], out_q=buf[1:5])
    with pytest.raises(DrkvError):                                       # every row written to the same place
        rope.apply(pos, x, out_q=buf[:1].expand(4, 2, 64))
    assert not buf.any()


@pytest.mark.gpu
def test_gradient_is_the_transpose(drkv_lib):
    """<R x, g> = <x, R^T g>, and R^T g against differences of <R x, g> (the operator is linear: exact up to rounding)."""
    import torch
    from deusridet_b200 import Rope
    kw = SCALINGS["ramp"]
    rope = Rope(head_dim=32, rotary_dim=24, dtype="f16", scaling="ramp", device=0, **kw)
    g = torch.Generator(device="cuda").manual_seed(9)
    pos = torch.tensor([0, 5, 70000], device="cuda", dtype=torch.int32)
    x, up = (torch.randn(3, 2, 32, generator=g, device="cuda").half() for _ in range(2))
    grad, _ = rope.apply(pos, up, inverse=True)
    freq, a = expected_frequencies(24, 1e4, "ramp", **kw)
    want, mag = rotate64(up.double().cpu().numpy(), pos.cpu().numpy(), freq, a, "halves", True)
    diff = np.zeros_like(want)
    for t in range(3):
        for h in range(2):
            for i in range(32):
                e = torch.zeros_like(x)
                e[t, h, i] = 1.0
                y, _ = rope.apply(pos, e)
                diff[t, h, i] = float((y.double() * up.double()).sum())
    # two entries of y, each rounded to fp16 (2^-11 relative, at most a), times |up|
    tol = 2.0 ** -11 * a * (mag + np.abs(up.double().cpu().numpy())) + 2.0 ** -11 * np.abs(want) + 1e-5
    assert (np.abs(diff - grad.double().cpu().numpy()) <= tol).all()
    assert (np.abs(want - grad.double().cpu().numpy()) <= tol).all()


@pytest.mark.gpu
def test_stream_and_graph(drkv_lib):
    """On a side stream, and captured: a replay reads the positions and rows of its own time."""
    import torch
    from deusridet_b200 import Rope
    rope = Rope(head_dim=128, dtype="bf16", device=0)
    freq, a = expected_frequencies(128, 1e4, "none")
    g = torch.Generator(device="cuda").manual_seed(4)
    pos = torch.zeros(9, device="cuda", dtype=torch.int32)
    q = torch.zeros(9, 4, 128, device="cuda", dtype=torch.bfloat16)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        rope.apply(pos, q, out_q=out, stream=torch.cuda.current_stream())
    for step in range(2):
        pos.copy_(torch.arange(9, device="cuda") + 1000 * step)
        q.copy_(torch.randn(9, 4, 128, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, pos, freq, a, "halves", False, torch.bfloat16)
