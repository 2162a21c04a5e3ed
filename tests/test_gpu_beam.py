"""beam_select and beam_reorder against numpy, bit-exact: totals are fp32 sums
whose roundings the definition fixes, so choice, order and score are too."""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


def select_oracle(x, cum, lse, allowed, k):
    """x: float32 [B, W, V]; allowed: bool [V], [B, W, V] or None."""
    b, w, v = x.shape
    with np.errstate(invalid="ignore"):
        total = cum[:, :, None] + (x - lse[:, :, None] if lse is not None else x)
    total = total.astype(np.float32)
    total[np.isnan(total)] = -np.inf
    if allowed is not None:
        total[~np.broadcast_to(allowed, total.shape)] = -np.inf
    total = total.reshape(b, w * v)
    place = np.argsort(-total, axis=1, kind="stable")[:, :k]
    scores = np.take_along_axis(total, place, 1)
    none = np.full((b, k), -np.inf, np.float32)
    tokens, parents = np.full((b, k), -1, np.int32), np.full((b, k), -1, np.int32)
    n = place.shape[1]
    ok = scores > -np.inf
    none[:, :n][ok] = scores[ok]
    tokens[:, :n][ok] = (place % v)[ok]
    parents[:, :n][ok] = (place // v)[ok]
    return none, tokens, parents


def run_select(gpu, x, cum, k, lse=None, allowed=None):
    import torch
    b = x.shape[0]
    out = (torch.full((b, k), 7.0, device="cuda"), torch.full((b, k), 7, device="cuda", dtype=torch.int32),
           torch.full((b, k), 7, device="cuda", dtype=torch.int32))
    gpu.beam_select(x, cum, *out, d_lse=lse, allowed=allowed)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in out]


def check(gpu, x, cum, k, lse=None, mask=None, allowed=None):
    host = lambda t: None if t is None else t.float().cpu().numpy()  # noqa: E731
    want = select_oracle(host(x), host(cum), host(lse), mask, k)
    got = run_select(gpu, x, cum, k, lse, allowed)
    for g, w, name in zip(got, want, ("scores", "tokens", "parents")):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5], g[g != w][:5], w[g != w][:5])


def _inputs(b, w, v, dtype, seed, pad=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(b, w, v + pad, device="cuda", generator=g).mul_(3).to(getattr(torch, dtype))[:, :, :v]
    cum = -10 * torch.rand(b, w, device="cuda", generator=g)
    return x, cum


def _bits(mask):
    words = np.zeros(mask.shape[:-1] + ((mask.shape[-1] + 31) // 32 * 32,), bool)
    words[..., :mask.shape[-1]] = mask
    return np.packbits(words, axis=-1, bitorder="little").view(np.int32)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("b,w,v,k", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 3, 511, 6), (3, 4, 513, 8), (1, 8, 4097, 16),
                                     (2, 5, 32001, 10), (1, 64, 1000, 128), (2, 2, 300, 256), (1, 1, 100003, 256),
                                     (4, 1, 70000, 1), (1, 300, 5, 7)])
def test_select(gpu, dtype, b, w, v, k):
    _say("beam", dtype, b, w, v, k)
    x, cum = _inputs(b, w, v, dtype, v)
    check(gpu, x, cum, k)
    import torch
    check(gpu, x, cum, k, lse=torch.logsumexp(x.float(), 2).contiguous())


@pytest.mark.parametrize("pad", [1, 3, 8])
def test_select_strides(gpu, pad):
    """Rows that start at every alignment."""
    _say("beam strides", pad)
    for dtype in ("float32", "bfloat16"):
        x, cum = _inputs(2, 5, 2000, dtype, pad, pad)
        check(gpu, x, cum, 9)
    x, cum = _inputs(2, 4, 1500, "float16", pad)
    check(gpu, x[:, ::2], cum[:, ::2].contiguous(), 5)


@pytest.mark.parametrize("density", [0.0, 0.001, 0.3, 1.0])
@pytest.mark.parametrize("v", [40, 5000, 70001, 140000])
def test_select_allowed(gpu, density, v):
    import torch
    _say("beam allowed", density, v)
    rng = np.random.default_rng(v)
    for dtype, pad in (("float32", 0), ("bfloat16", 1)):
        x, cum = _inputs(2, 3, v, dtype, v, pad)
        mask = rng.random(v) < density
        ids = np.nonzero(mask)[0].astype(np.uint32)
        for thr in (gpu.PROMOTE_ALL, gpu.PROMOTE_KEEP_DEFAULT):
            g = gpu.upload_from_ids(ids, v, thr)
            check(gpu, x, cum, 12, mask=mask, allowed=g)
            gpu.free(g)
        check(gpu, x, cum, 12, mask=mask, allowed=torch.from_numpy(_bits(mask)).cuda())
        each = rng.random((2, 3, v)) < density
        each[0, 1] = False  # a beam that may not go on
        check(gpu, x, cum, 12, mask=each, allowed=torch.from_numpy(_bits(each)).cuda())


def test_select_from_batched_bitmaps(gpu):
    """One set per beam, kept as a batch of bitmaps and decompressed for the step."""
    import torch
    _say("beam from a batch of bitmaps")
    v, b, w = 4096, 1, 3
    rng = np.random.default_rng(9)
    sets = [np.sort(rng.choice(v, n, replace=False)).astype(np.uint16) for n in (5, 900, 64)]
    batch = gpu.upload_batch([[(0, gpu.TC_ARRAY, len(s), s)] for s in sets])
    # a batch's bitmaps end with their last key's container: room for 65536 ids each
    words = torch.zeros(3, 1024, dtype=torch.int64, device="cuda")
    gpu.batch_decompress(batch, words, 1024)
    bits = words.view(torch.int32).view(b, w, 2048)[:, :, :v // 32].contiguous()
    mask = np.zeros((b, w, v), bool)
    for i, s in enumerate(sets):
        mask[0, i, s] = True
    x, cum = _inputs(b, w, v, "bfloat16", 3)
    check(gpu, x, cum, 20, mask=mask, allowed=bits)
    gpu.free_batch(batch)


def test_select_ties(gpu):
    """Equal totals go to the lowest place, within a beam, over beams, and where every total is the same."""
    import torch
    _say("beam ties")
    x = torch.zeros(2, 4, 3001, device="cuda")
    cum = torch.zeros(2, 4, device="cuda")
    check(gpu, x, cum, 20)
    check(gpu, x.bfloat16(), cum, 256)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(0, 3, (2, 4, 30001), device="cuda", generator=g).float()
    check(gpu, x, cum, 50)
    x[:, 1:, ::7] = -0.0
    x[:, 0] = 0.0
    check(gpu, x.clamp(max=0), cum, 30)
    # the same totals by different ways
    x = torch.zeros(1, 2, 600, device="cuda")
    x[0, 0, 5] = x[0, 1, 3] = 4.0
    check(gpu, x, torch.tensor([[1.0, 1.0]], device="cuda"), 3)


def test_select_ordered_scores(gpu):
    """Scores that rise or fall along the vocabulary: all the best in one place, or the best always last."""
    import torch
    _say("beam ordered")
    for v in (5000, 200000):
        up = torch.arange(v, device="cuda").float().div_(1024)
        for x in (up, -up):
            check(gpu, x[None, None].repeat(1, 2, 1).contiguous(), torch.zeros(1, 2, device="cuda"), 100)


def test_select_no_candidates(gpu):
    import torch
    _say("beam without candidates")
    inf = float("inf")
    x, cum = _inputs(3, 4, 1000, "float32", 5)
    cum[0] = -inf
    cum[1, 1:] = -inf
    x[2, 0] = float("nan")
    x[2, 1, :500] = -inf
    x[2, 2, 7] = inf
    cum[2, 3] = float("nan")
    check(gpu, x, cum, 8)
    x[:] = -inf
    x[1, 0, 999], x[1, 0, 3] = 1.0, 0.5
    check(gpu, x, cum, 8)


def test_select_many_over_the_bound(gpu):
    """Thousands of equal totals just over the bound of the first pass."""
    import torch
    _say("beam many candidates")
    x = torch.full((1, 3, 150000), -5.0, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    x[0, torch.randint(0, 3, (20000,), device="cuda", generator=g),
      torch.randint(0, 150000, (20000,), device="cuda", generator=g)] = 1.0
    x[0, 2, 149999] = 2.0
    check(gpu, x, torch.zeros(1, 3, device="cuda"), 256)
    check(gpu, x.half(), torch.zeros(1, 3, device="cuda"), 100)


# ---- reorder ---------------------------------------------------------------------
@pytest.mark.parametrize("b,w,v,k", [(3, 8, 1507, 8), (2, 5, 5614, 10), (2, 2, 1025, 2), (4, 4, 16468, 8),
                                     (1, 3, 30000, 64), (2, 1, 70000, 256), (1, 6, 2047, 200)])
def test_select_from_few_groups(gpu, b, w, v, k):
    """Few pieces of the vocabulary to bound the answer by: as they come, equal, one lane's, and few allowed."""
    import torch
    _say("beam few groups", b, w, v, k)
    x, cum = _inputs(b, w, v, "bfloat16", 31)
    check(gpu, x, cum, k)
    mask = np.zeros(v, bool)
    mask[v // 3:v // 3 + 90] = True
    bits = torch.from_numpy(_bits(mask)).cuda()
    check(gpu, x, cum, k, mask=mask, allowed=bits)
    x[:, :, 8:16] += 50.0  # the best are neighbours: a lane has several of them
    check(gpu, x, cum, k)
    x[:, :, ::3] = float("nan")
    x[:, :, 1::5] = float("-inf")
    check(gpu, x, cum, k)
    check(gpu, torch.zeros_like(x), torch.zeros_like(cum), k)


@pytest.mark.parametrize("dtype,shape", [("bfloat16", (40, 8, 64)), ("int32", (17,)), ("uint8", (5, 3)), ("float32", (1,)),
                                         ("float16", (3, 70000)), ("int64", (33, 2))])
@pytest.mark.parametrize("lengths", [False, True])
def test_reorder(gpu, dtype, shape, lengths):
    import torch
    _say("reorder", dtype, shape, lengths)
    b, w, k = 3, 4, 6
    g = torch.Generator(device="cuda").manual_seed(7)
    new = lambda n: torch.randint(0, 100, (b, n) + shape, device="cuda", generator=g).to(getattr(torch, dtype))  # noqa: E731
    src, dst = new(w), new(k)
    parents = torch.randint(0, w, (b, k), device="cuda", generator=g).to(torch.int32)
    parents[1, 2], parents[2, 5] = -1, w
    length = torch.randint(0, shape[0] + 3, (b, w), device="cuda", generator=g).to(torch.int32) if lengths else None
    if lengths:
        length[0, 0] = -4
    want = dst.clone()
    for i in range(b):
        for j in range(k):
            p = int(parents[i, j])
            if 0 <= p < w:
                n = shape[0] if length is None else min(shape[0], max(0, int(length[i, p])))
                want[i, j, :n] = src[i, p, :n]
    gpu.beam_reorder(src, parents, dst, length)
    torch.cuda.synchronize()
    assert torch.equal(dst, want)


def test_reorder_more_rows_than_a_grid_has(gpu):
    import torch
    _say("reorder 70000 rows")
    src = torch.arange(70000 * 2 * 4, device="cuda", dtype=torch.int32).view(35000, 4, 4)
    parents = torch.randint(0, 4, (35000, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    dst = torch.zeros(35000, 2, 4, device="cuda", dtype=torch.int32)
    gpu.beam_reorder(src, parents.to(torch.int32), dst)
    torch.cuda.synchronize()
    assert torch.equal(dst, torch.gather(src, 1, parents[:, :, None].expand(-1, -1, 4)))


def test_refusals(gpu):
    import torch
    _say("beam refusals")
    x, cum = _inputs(2, 3, 100, "float32", 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    out = lambda k: dict(d_out_scores=torch.zeros(2, k, device="cuda"), d_out_tokens=torch.zeros(2, k, **i32),  # noqa: E731
                         d_out_parents=torch.zeros(2, k, **i32))
    ok = dict(d_scores=x, d_cum=cum, **out(4))
    gpu.beam_select(**ok)
    for bad, code in ((dict(d_scores=x.double()), gpu.CR_ERR_INVALID), (dict(d_cum=cum[:1]), gpu.CR_ERR_INVALID),
                      (dict(d_cum=cum.half()), gpu.CR_ERR_INVALID), (dict(d_scores=x.transpose(1, 2)), gpu.CR_ERR_INVALID),
                      (dict(d_lse=cum[:, :2].contiguous()), gpu.CR_ERR_INVALID),
                      (dict(allowed=torch.zeros(5, **i32)), gpu.CR_ERR_INVALID),
                      (dict(d_out_tokens=torch.zeros(2, 3, **i32)), gpu.CR_ERR_INVALID),
                      (out(257), gpu.CR_ERR_UNSUPPORTED)):
        with pytest.raises(gpu.CrError) as e:
            gpu.beam_select(**{**ok, **bad})
        assert e.value.code == code, bad.keys()
    s = torch.zeros(2, 3, 8, device="cuda")
    p = torch.zeros(2, 3, **i32)
    for bad in (dict(d_dst=s), dict(d_dst=torch.zeros(2, 4, 8, device="cuda")), dict(d_dst=s.half()),
                dict(d_parents=p.long()), dict(d_len=p[:1]), dict(d_dst=s.clone().transpose(0, 1))):
        with pytest.raises(gpu.CrError):
            gpu.beam_reorder(**{**dict(d_src=s, d_parents=p, d_dst=s.clone()), **bad})
    torch.cuda.synchronize()
