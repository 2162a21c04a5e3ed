"""paged_rotary against the formula in 64 bits.

The bar of a turned element of x, y and magnitude m, with u the type's unit
roundoff: the result is rounded once (u |want|; f16 below its normal range by
2^-25 at most).  An angle within an eighth of a turn is rounded once (2^-24 of
0.79) and its series' terms sum to another 2^-23 or less, with 2^-29 left out, so
that cosine and sine are off by less than 2^-22.5; they are rounded once more with
m, and two fp32 products and their sum add 2^-23 of m (|x| + |y|): 2^-21 of that in
all.  The turns themselves, in 64 bits, are off by 2^-51 of up to 2^22.
"""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def _say(*a):
    print("CASE", *a, flush=True)


def _host(t):
    return t.double().cpu().numpy()


def turned(x, positions, freqs, m, interleaved):
    """(want, what |x| + |y| of each element's pair is): float64 [T, heads, dim]."""
    rot = 2 * len(freqs)
    a = positions.astype(np.float64)[:, None] * freqs
    c, s = np.cos(a)[:, None] * m, np.sin(a)[:, None] * m
    i = np.arange(rot // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    want, size = x.copy(), np.zeros_like(x)
    want[..., first] = x[..., first] * c - x[..., second] * s
    want[..., second] = x[..., second] * c + x[..., first] * s
    size[..., first] = size[..., second] = abs(m) * (np.abs(x[..., first]) + np.abs(x[..., second]))
    return want, size


def check_turned(got, x, positions, freqs, m, interleaved, dtype):
    want, size = turned(x, positions, freqs, m, interleaved)
    tol = np.where(size > 0, 1.01 * (U[dtype] * np.abs(want) + 2.0 ** -21 * size +
                                     (2.0 ** -25 if dtype == "float16" else 0)), 0.0)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)


def check(gpu, dtype, tokens, heads, kv_heads, dim, rot, interleaved, page=16, layout="plain", far=5000, m=1.0,
          in_place=False, hole=False, seed=0, stream=None, scaling=None):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    pages = -(-tokens // page) + 3

    def rows(h):
        if layout == "padded":
            return rnd(tokens, h + 1, dim + 8).to(dt)[:, 1:, :dim]
        if layout == "odd":  # rows that begin anywhere
            return rnd(tokens, h, dim + 1).to(dt)[..., 1:]
        if layout == "heads first":
            return rnd(h, tokens, dim).to(dt).transpose(0, 1)
        return rnd(tokens, h, dim).to(dt)

    def cache():
        if layout == "heads first":
            return torch.full((pages, kv_heads, page, dim), 3.0, device="cuda").to(dt).transpose(1, 2)
        if layout == "odd":
            return torch.full((pages, page, kv_heads, dim + 1), 3.0, device="cuda").to(dt)[..., 1:]
        return torch.full((pages, page, kv_heads, dim), 3.0, device="cuda").to(dt)

    q, k, v, kc, vc = rows(heads) if heads else None, rows(kv_heads), rows(kv_heads), cache(), cache()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    if hole:
        slots[::3] = -1
        slots[1::7] = pages * page
    positions = torch.randint(-far, far + 1, (tokens,), device="cuda", generator=g).to(torch.int32)
    freqs, magnitude = gpu.rotary_frequencies(rot, scaling=scaling, factor=8.0 if scaling else 1.0)
    q0 = _host(q) if heads else None
    out = None if not heads else q if in_place else torch.full_like(q, 7.0)
    gpu.paged_rotary(k, v, positions, freqs, slots, kc, vc, d_q=q, d_q_out=None if in_place else out,
                     interleaved=interleaved, magnitude=m * magnitude, stream=stream)
    torch.cuda.synchronize()
    f, p, mm = freqs.cpu().numpy(), positions.cpu().numpy(), float(np.float32(m * magnitude))
    if heads:
        check_turned(_host(out), q0, p, f, mm, interleaved, dtype)
        if not in_place:
            assert np.array_equal(_host(q), q0)
    at = slots.cpu().numpy()
    there = (at >= 0) & (at < pages * page)
    kc, vc = (np.array(_host(t)).reshape(-1, kv_heads, dim) for t in (kc, vc))
    check_turned(kc[at[there]], _host(k)[there], p[there], f, mm, interleaved, dtype)
    assert np.array_equal(vc[at[there]], _host(v)[there])
    rest = np.ones(pages * page, bool)
    rest[at[there]] = False
    assert np.all(kc[rest] == 3.0) and np.all(vc[rest] == 3.0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", [
    (1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (64, 32, 8, 128, 64), (37, 6, 2, 80, 20), (7, 3, 3, 96, 24), (300, 4, 1, 192, 48),
    (5, 5, 5, 256, 256), (129, 2, 1, 72, 66), (3, 2, 2, 7, 6), (2, 1, 1, 2, 2), (515, 1, 1, 8, 8), (9, 2, 1, 64, 0)])
def test_rotary(gpu, dtype, interleaved, tokens, heads, kv_heads, dim, rot):
    _say("rotary", dtype, interleaved, tokens, heads, kv_heads, dim, rot)
    check(gpu, dtype, tokens, heads, kv_heads, dim, rot, interleaved, seed=tokens + dim)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["padded", "odd", "heads first"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rotary_strides(gpu, dtype, layout, interleaved):
    _say("rotary strides", dtype, layout, interleaved)
    check(gpu, dtype, 45, 6, 2, 64, 32, interleaved, layout=layout)


@pytest.mark.parametrize("what", [dict(in_place=True), dict(hole=True), dict(m=-0.5), dict(far=2 ** 24), dict(page=1),
                                  dict(page=512), dict(scaling="linear"), dict(scaling="base"), dict(scaling="parts")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_edges(gpu, interleaved, what):
    _say("rotary", interleaved, what)
    check(gpu, "float32", 70, 4, 2, 96, 64, interleaved, **what)
    check(gpu, "float16", 70, 4, 2, 96, 64, interleaved, **what)


def test_keys_alone(gpu):
    _say("rotary without queries")
    check(gpu, "bfloat16", 33, 0, 4, 128, 128, False)


def test_no_tokens(gpu):
    import torch
    _say("rotary without tokens")
    k = torch.zeros(0, 2, 64, device="cuda")
    c = torch.full((2, 16, 2, 64), 3.0, device="cuda")
    gpu.paged_rotary(k, k, torch.zeros(0, dtype=torch.int32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda"),
                     torch.zeros(0, dtype=torch.int64, device="cuda"), c, c.clone())
    torch.cuda.synchronize()
    assert torch.all(c == 3.0)


def test_another_stream(gpu):
    import torch
    _say("rotary on another stream")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check(gpu, "bfloat16", 200, 8, 2, 128, 128, False, stream=s)


def test_many_tokens(gpu):
    _say("rotary of many tokens")
    check(gpu, "bfloat16", 5003, 3, 1, 128, 128, False, page=64)
    check(gpu, "float16", 20011, 1, 1, 64, 32, True, page=128)


def test_scores_go_by_the_distance(gpu):
    """Turned queries and keys meet as their distance says: moving both by the same positions changes no product."""
    import torch
    _say("rotary distances")
    freqs, _ = gpu.rotary_frequencies(64)
    q, k = torch.randn(1, 1, 64, device="cuda"), torch.randn(1, 1, 64, device="cuda")
    q, k = q.expand(9, 1, 64).contiguous(), k.expand(9, 1, 64).contiguous()
    at = torch.arange(9, dtype=torch.int32, device="cuda") * 1000
    kc, vc = torch.zeros(9, 1, 1, 64, device="cuda"), torch.zeros(9, 1, 1, 64, device="cuda")
    slots = torch.arange(9, device="cuda")
    q1, q2 = torch.empty_like(q), torch.empty_like(q)
    gpu.paged_rotary(k, k, at, freqs, slots, kc, vc, d_q=q, d_q_out=q1)
    k1 = kc.clone().view(9, 64)
    gpu.paged_rotary(k, k, at + 77, freqs, slots, kc, vc, d_q=q, d_q_out=q2)
    torch.cuda.synchronize()
    same = (q1.view(9, 64).double() * k1.double()).sum(1)
    size = float(q.double().norm(dim=2).max() * k.double().norm(dim=2).max())
    assert (same - same[0]).abs().max() < 2.0 ** -19 * size  # two rows, each off by 2^-20 of its length or less
    far = (q2.view(9, 64).double() * kc.view(9, 64).double()).sum(1)
    assert (far - same).abs().max() < 2.0 ** -19 * size
