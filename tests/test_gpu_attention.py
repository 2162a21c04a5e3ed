"""paged_attention against the formula in 64 bits.

The bar of an output element, with u the type's unit roundoff (2^-8 bf16, 2^-11
f16) and w = sum_j p_j |v_j| over the normalised probabilities p: the result is
rounded once (u |o|) and each probability is rounded once before it meets its
value (u w; below f16's normal range by 2^-25 at most, n 2^-25 max|v|).  Scores
are fp32 sums of exact products: their error moves a probability by at most
(dim + 8) 2^-23 |scale| sum|q k| relative, counted twice (numerator and sum), as
do fp32 sums over n keys by n 2^-24.  An lse is off by the same score error and
by 2^-22 of itself and of log n.
"""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _say(*a):
    print("CASE", *a, flush=True)


class Problem:
    """Requests over a paged cache, the pages scattered and the unused ones full of NaN."""

    def __init__(self, dtype, new, kv, heads, kv_heads, dim, page, seed=0, spread=2.0, layout="plain", density=None,
                 causal=True):
        import torch
        self.torch, self.dtype, self.page, self.causal = torch, dtype, page, causal
        self.new, self.kv = list(new), list(kv)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        dt = getattr(torch, dtype)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        held = [-(-max(0, x) // page) for x in kv]
        self.cols = max(1, max(held, default=1))
        pages = sum(held) + 3
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(kv), self.cols), -1, dtype=torch.int32, device="cuda")
        at = 0
        for r, n in enumerate(held):
            self.table[r, :n] = order[at:at + n]
            at += n
        def cache():
            if layout == "heads first":
                return rnd(pages, kv_heads, page, dim).to(dt).transpose(1, 2)
            if layout == "padded":
                return rnd(pages, page, kv_heads, dim + 16).to(dt)[..., 8:8 + dim]
            return rnd(pages, page, kv_heads, dim).to(dt)
        self.kc, self.vc = cache(), cache()
        self.kc[order[at:].long()] = float("nan")
        self.vc[order[at:].long()] = float("nan")
        for r, n in enumerate(held):  # what lies behind a request's last token is not read into its answer
            if n and kv[r] % page:
                self.kc[self.table[r, n - 1].long(), kv[r] % page:] = float("nan")
                self.vc[self.table[r, n - 1].long(), kv[r] % page:] = float("nan")
        total = sum(new)
        if layout == "heads first":
            self.q = (rnd(heads, total, dim) * spread).to(dt).transpose(0, 1)
        elif layout == "padded":
            self.q = (rnd(total, heads + 2, dim + 8) * spread).to(dt)[:, 1:1 + heads, :dim]
        else:
            self.q = (rnd(total, heads, dim) * spread).to(dt)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        self.kv_len = torch.tensor(kv, **i32)
        self.visible = None
        if density is not None:
            self.visible = (torch.rand(pages * page, device="cuda", generator=g) < density)
            self.sel = torch.full((len(kv), self.cols * page), -1, **i32)
            self.sel_len, self.limits = torch.zeros(len(kv), **i32), torch.zeros(total, **i32)

    def run(self, gpu, scale=None, **kw):
        torch = self.torch
        selection = None
        if self.visible is not None:
            words = self.visible.cpu().numpy()
            ids = np.nonzero(words)[0].astype(np.uint32)
            g = gpu.upload_from_ids(ids, len(words))
            gpu.paged_select(g, self.table, self.starts, self.kv_len, self.page, self.sel, self.sel_len, self.limits,
                             self.kc.shape[0])
            selection = (self.sel, self.sel_len, self.limits)
        out = torch.full((sum(self.new) + 2, self.heads, self.dim), 7.0, device="cuda", dtype=self.q.dtype)
        lse = torch.full((sum(self.new), self.heads), 7.0, device="cuda")
        gpu.paged_attention(self.q, self.kc, self.vc, self.table, self.starts, self.kv_len, out[:sum(self.new)],
                            scale=scale, causal=self.causal, d_lse=lse, selection=selection, **kw)
        torch.cuda.synchronize()
        if selection is not None:
            gpu.free(g)
        assert torch.all(out[sum(self.new):] == 7.0), "written past the last token"
        return out[:sum(self.new)].float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)

    def check(self, gpu, scale=None, **kw):
        out, lse = self.run(gpu, scale, **kw)
        scale = self.dim ** -0.5 if scale is None else scale
        u, group = U[self.dtype], self.heads // self.kv_heads
        host = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
        q, table = host(self.q), self.table.cpu().numpy()
        kc, vc = host(self.kc), host(self.vc)
        visible = None if self.visible is None else self.visible.cpu().numpy()
        at = 0
        for n, kv, row in zip(self.new, self.kv, table):
            pos = np.arange(max(0, kv))
            page, off = row[pos // self.page], pos % self.page
            if visible is not None:
                keep = visible[page * self.page + off]
                pos, page, off = pos[keep], page[keep], off[keep]
            for h in range(self.heads if n else 0):
                k, v = kc[page, off, h // group], vc[page, off, h // group]
                for i in range(n):
                    see = pos <= kv - n + i if self.causal else pos >= 0
                    o, z = out[at + i, h], lse[at + i, h]
                    if not see.any():
                        assert np.all(o == 0) and z == -np.inf, (at + i, h)
                        continue
                    s = scale * (k[see] @ q[at + i, h])
                    ds = (self.dim + 8) * 2.0 ** -23 * abs(scale) * (np.abs(k[see]) @ np.abs(q[at + i, h])).max()
                    m = s.max()
                    p = np.exp(s - m)
                    z0 = m + np.log(p.sum())
                    p /= p.sum()
                    o0, w = p @ v[see], p @ np.abs(v[see])
                    c = int(see.sum())
                    tiny = c * 2.0 ** -25 * np.abs(v[see]).max() if self.dtype == "float16" else 0.0
                    tol = 1.01 * (u * np.abs(o0) + u * w + tiny + (2 * ds + c * 2.0 ** -24 + 2.0 ** -20) * w)
                    assert np.all(np.abs(o - o0) <= tol), (at + i, h, np.max(np.abs(o - o0) / tol))
                    assert abs(z - z0) <= ds + 2.0 ** -22 * (abs(z0) + np.log(c) + 2) + c * 2.0 ** -24, (at + i, h, z, z0)
            at += n


# new, kv, heads, key heads, dim, page
SHAPES = {
    "one token, one key": ([1], [1], 1, 1, 64, 16),
    "short context": ([1], [37], 8, 2, 128, 16),
    "decode ragged": ([1, 1, 1, 1, 1], [1, 16, 17, 300, 1025], 8, 2, 128, 16),
    "decode mha": ([1, 1, 1], [63, 64, 65], 5, 5, 64, 32),
    "decode wide group": ([1, 1], [200, 129], 24, 1, 128, 8),
    "decode group 33": ([1], [150], 33, 1, 64, 16),
    "no tokens between": ([1, 0, 2, 0], [40, 33, 70, 0], 4, 4, 64, 16),
    "a few tokens": ([4, 3, 5], [260, 3, 131], 16, 4, 128, 16),
    "chunk": ([130, 1, 64], [400, 77, 64], 4, 2, 128, 16),
    "prompt": ([257], [257], 4, 1, 64, 64),
    "prompt group 3": ([100, 45], [100, 300], 6, 2, 96, 16),
    "dims 8": ([3, 40], [50, 40], 4, 2, 8, 16),
    "dims 80": ([1, 70], [333, 70], 4, 2, 80, 16),
    "dims 192": ([1, 70], [129, 200], 4, 2, 192, 16),
    "dims 256": ([2, 90], [97, 150], 4, 2, 256, 16),
    "pages of one": ([1, 20], [70, 66], 2, 1, 64, 1),
    "pages longer than the context": ([1, 20], [70, 66], 2, 2, 64, 1024),
    "more tokens than positions": ([9, 70], [5, 40], 2, 1, 64, 16),
    "negative length": ([2, 1], [-3, 20], 2, 1, 64, 16),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("what", SHAPES)
def test_attention(gpu, dtype, what):
    _say("attention", dtype, what)
    Problem(dtype, *SHAPES[what], seed=len(what)).check(gpu)


@pytest.mark.parametrize("density", [0.0, 0.02, 0.4, 1.0])
@pytest.mark.parametrize("what", ["decode ragged", "a few tokens", "chunk", "prompt group 3", "pages of one",
                                  "more tokens than positions"])
def test_attention_over_a_selection(gpu, what, density):
    _say("attention selection", what, density)
    Problem("float16", *SHAPES[what], seed=3, density=density).check(gpu)


@pytest.mark.parametrize("density", [None, 0.3])
@pytest.mark.parametrize("what", ["decode ragged", "chunk", "more tokens than positions"])
def test_attention_not_causal(gpu, what, density):
    _say("attention not causal", what, density)
    Problem("bfloat16", *SHAPES[what], seed=4, density=density, causal=False).check(gpu)


@pytest.mark.parametrize("layout", ["heads first", "padded"])
@pytest.mark.parametrize("what", ["decode ragged", "chunk", "dims 80"])
def test_attention_strides(gpu, what, layout):
    _say("attention strides", what, layout)
    Problem("bfloat16", *SHAPES[what], seed=5, layout=layout).check(gpu)


@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 1.0), (1.0, 8.0), (1e-3, 1.0)])
@pytest.mark.parametrize("what", ["decode ragged", "chunk"])
def test_attention_scales(gpu, what, scale, spread):
    """Scores that are all alike, turned round, and hundreds apart (one key takes everything)."""
    _say("attention scale", what, scale)
    Problem("float16", *SHAPES[what], seed=6, spread=spread).check(gpu, scale=scale)


@pytest.mark.parametrize("hints", [dict(max_new=1, max_kv=1), dict(max_new=5000, max_kv=1 << 20), dict(max_kv=200)])
@pytest.mark.parametrize("what", ["decode ragged", "chunk"])
def test_hints_do_not_change_the_answer(gpu, what, hints):
    _say("attention hints", what, hints)
    Problem("bfloat16", *SHAPES[what], seed=7).check(gpu, **hints)


@pytest.mark.parametrize("new,kv", [([1], [20011]), ([1, 1], [5000, 12345]), ([17], [9000]), ([1], [65536])])
def test_attention_long_contexts(gpu, new, kv):
    _say("attention long", new, kv)
    Problem("bfloat16", new, kv, 8, 2, 128, 16, seed=8).check(gpu)
    Problem("float16", new, kv, 4, 4, 64, 32, seed=9, density=0.2).check(gpu)


def test_rising_scores(gpu):
    """Each key's score beats all before it, by little and by much: the running maximum moves at every key."""
    import torch
    for step in (0.02, 1.5):
        for new, kv in (([1], [700]), ([90], [300])):
            _say("attention rising", step, kv)
            p = Problem("float16", new, kv, 2, 1, 64, 16, seed=10)
            p.q[:] = 0
            p.q[:, :, 0] = 1.0
            row = p.table[0].long()
            pos = torch.arange(kv[0], device="cuda")
            p.kc[row[pos // 16], pos % 16, :, 0] = (pos * step).half()[:, None]
            p.check(gpu, scale=1.0)


def test_infinite_and_nan_values_where_nothing_looks(gpu):
    """Keys and values after a token's position hold inf and NaN: earlier tokens do not see them."""
    for bad in (float("inf"), float("-inf"), float("nan")):
        _say("attention", bad, "behind the causal limit")
        p = Problem("bfloat16", [5], [105], 4, 2, 64, 16, seed=11)
        whole, _ = p.run(__import__("curoaring"))
        for pos in (103, 104):
            page = p.table[0, pos // 16].long()
            p.kc[page, pos % 16] = bad
            p.vc[page, pos % 16] = bad
        out, lse = p.run(__import__("curoaring"))
        assert np.array_equal(out[:3], whole[:3]) and np.all(np.isfinite(lse[:3]))


def test_pages_outside_the_cache_are_not_seen(gpu):
    _say("attention with pages outside the cache")
    p = Problem("bfloat16", [1, 40], [100, 90], 4, 2, 64, 16, seed=12)
    p.table[0, 2], p.table[1, 1] = -1, p.kc.shape[0]
    seen = p.run(gpu)
    # the same with a selection that leaves these positions out
    ref = Problem("bfloat16", [1, 40], [100, 90], 4, 2, 64, 16, seed=12, density=1.0)
    keep = ref.visible.clone()
    for r, c in ((0, 2), (1, 1)):
        page = int(ref.table[r, c])
        keep[page * 16:page * 16 + 16] = False
    ref.visible = keep
    want = ref.run(gpu)
    assert np.allclose(seen[0], want[0], rtol=2.0 ** -6, atol=2.0 ** -6) and np.allclose(seen[1], want[1], rtol=1e-5)


def test_tokens_in_no_request_get_zeros(gpu):
    import torch
    _say("attention tokens in no request")
    p = Problem("float16", [3, 2], [50, 40], 2, 1, 64, 16, seed=13)
    want, want_lse = p.run(gpu)
    q = torch.cat([p.q, torch.ones_like(p.q)])
    out, lse = torch.full_like(q, 7.0), torch.full((10, 2), 7.0, device="cuda")
    gpu.paged_attention(q, p.kc, p.vc, p.table, p.starts, p.kv_len, out, d_lse=lse)
    torch.cuda.synchronize()
    assert np.array_equal(out[:5].float().cpu().numpy(), want) and np.array_equal(lse[:5].cpu().numpy(), want_lse)
    assert torch.all(out[5:] == 0) and torch.all(lse[5:] == float("-inf"))


def test_no_requests(gpu):
    import torch
    _say("attention without requests")
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.ones(3, 2, 64, device="cuda").half()
    out = torch.full_like(q, 7.0)
    kc = torch.zeros(2, 16, 1, 64, device="cuda").half()
    gpu.paged_attention(q, kc, kc.clone(), torch.zeros(0, 1, **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), out)
    torch.cuda.synchronize()
    assert torch.all(out == 0)


def test_two_runs_give_the_same_bits(gpu):
    _say("attention twice")
    for what in ("decode ragged", "chunk", "a few tokens"):
        p = Problem("bfloat16", *SHAPES[what], seed=14)
        a, b = p.run(gpu), p.run(gpu)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_another_stream(gpu):
    import torch
    _say("attention on another stream")
    p = Problem("bfloat16", *SHAPES["decode ragged"], seed=15)
    want, _ = p.run(gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(p.q)
    with torch.cuda.stream(s):
        out.fill_(3.0)
        gpu.paged_attention(p.q, p.kc, p.vc, p.table, p.starts, p.kv_len, out, stream=s)
    s.synchronize()
    assert np.array_equal(out.float().cpu().numpy(), want)


def test_offsets_past_32_bits(gpu):
    """A cache whose last pages lie beyond 2^32 elements."""
    import torch
    _say("attention in a cache past 2^32 elements")
    p = Problem("float16", [1, 33], [200, 150], 8, 8, 128, 16, seed=16)
    want, want_lse = p.run(gpu)
    pages = (1 << 32) // (16 * 8 * 128) + 64
    used = p.kc.shape[0]
    for name in ("kc", "vc"):
        small = getattr(p, name)
        big = torch.empty(pages, 16, 8, 128, device="cuda", dtype=torch.float16)
        big[pages - used:] = small
        setattr(p, name, big)
    p.table[p.table >= 0] += pages - used
    out, lse = p.run(gpu)
    assert np.array_equal(out, want) and np.array_equal(lse, want_lse)


def test_refusals(gpu):
    import torch
    _say("attention refusals")
    p = Problem("float16", [2], [40], 4, 2, 64, 16)
    ok = dict(d_q=p.q, d_k_cache=p.kc, d_v_cache=p.vc, d_table=p.table, d_starts=p.starts, d_kv_len=p.kv_len,
              d_out=torch.empty_like(p.q))
    gpu.paged_attention(**ok)
    torch.cuda.synchronize()
    wide = torch.zeros(2, 4, 264, device="cuda").half()
    wide_c = torch.zeros(3, 16, 2, 264, device="cuda").half()
    odd = torch.zeros(2 * 4 * 64 + 1, device="cuda").half()[1:].view(2, 4, 64)
    for bad, code in ((dict(d_q=p.q.float(), d_out=p.q.float()), gpu.CR_ERR_INVALID),
                      (dict(d_q=p.q[:, :3], d_out=torch.empty_like(p.q[:, :3])), gpu.CR_ERR_INVALID),
                      (dict(d_q=p.q[:, :, :32]), gpu.CR_ERR_INVALID),
                      (dict(d_out=ok["d_out"][:1]), gpu.CR_ERR_INVALID),
                      (dict(d_v_cache=p.vc[:2]), gpu.CR_ERR_INVALID),
                      (dict(d_k_cache=p.kc[:, :12], d_v_cache=p.vc[:, :12]), gpu.CR_ERR_INVALID),
                      (dict(d_table=p.table.long()), gpu.CR_ERR_INVALID),
                      (dict(d_starts=p.starts[:1]), gpu.CR_ERR_INVALID),
                      (dict(d_kv_len=p.kv_len.long()), gpu.CR_ERR_INVALID),
                      (dict(d_lse=torch.zeros(2, 3, device="cuda")), gpu.CR_ERR_INVALID),
                      (dict(selection=(p.table, p.kv_len, p.kv_len)), gpu.CR_ERR_INVALID),
                      (dict(d_q=wide, d_out=wide.clone(), d_k_cache=wide_c, d_v_cache=wide_c), gpu.CR_ERR_UNSUPPORTED),
                      (dict(d_q=wide[..., :60], d_out=wide[..., :60].clone(), d_k_cache=wide_c[..., :60],
                            d_v_cache=wide_c[..., :60]), gpu.CR_ERR_UNSUPPORTED),
                      (dict(d_q=odd), gpu.CR_ERR_UNSUPPORTED),
                      (dict(d_k_cache=p.kc.float(), d_v_cache=p.vc.float(), d_q=p.q.float(), d_out=p.q.float()),
                       gpu.CR_ERR_UNSUPPORTED)):
        with pytest.raises(gpu.CrError) as e:
            gpu.paged_attention(**{**ok, **bad})
        assert e.value.code == code, bad.keys()


@pytest.mark.parametrize("hints", [{}, dict(max_kv=20000), dict(max_new=64), dict(max_new=64, max_kv=20000)])
def test_more_requests_than_a_wave_has_lanes(gpu, hints):
    """Over 64 requests, some without tokens or keys, by either kernel, with their keys cut into ranges or not."""
    _say("attention of 150 requests", hints)
    rng = np.random.default_rng(17)
    new = rng.integers(0, 4, 150).tolist()
    kv = [int(rng.integers(0, 300)) for _ in new]
    kv[77], new[77] = 2500, 3
    Problem("bfloat16", new, kv, 2, 1, 64, 16, seed=18).check(gpu, **hints)


@pytest.mark.parametrize("density", [None, 0.3])
@pytest.mark.parametrize("hints", [{}, dict(max_kv=5000), dict(max_new=1, max_kv=5000)])
def test_long_and_short_requests(gpu, hints, density):
    """One long request among short ones: some tiles are cut into ranges and others are whole."""
    _say("attention of long and short requests", hints, density)
    Problem("float16", [40, 3, 1, 0, 70], [4700, 30, 1, 9, 90], 4, 2, 96, 16, seed=19, density=density).check(gpu, **hints)


@pytest.mark.parametrize("dim", [64, 80, 128, 200])
@pytest.mark.parametrize("new,kv", [([1], [300]), ([2], [9000]), ([70], [200])])
def test_scores_that_are_not_finite(gpu, new, kv, dim):
    """A score of -inf takes no part, one of +inf or NaN makes the answers that see it NaN, and no others."""
    import torch
    shape, at = (new, kv, 4, 2, dim, 16), kv[0] - new[0] - 5
    p = Problem("bfloat16", *shape, seed=16)
    ref = Problem("bfloat16", *shape, seed=16, density=1.0)
    slot = int(p.table[0, at // 16]) * 16 + at % 16
    ref.visible = torch.ones_like(ref.visible)
    ref.visible[slot] = False
    for x in (p, ref):
        x.q[:, 0::2, 0], x.q[:, 1::2, 0] = 1.0, -1.0
    _say("attention infinite score", new, kv, dim)
    ref.check(gpu)
    want, want_lse = ref.run(gpu)
    p.kc[slot // 16, slot % 16, :, 0] = float("-inf")
    out, lse = p.run(gpu)
    assert np.allclose(out[:, 0::2], want[:, 0::2], rtol=2.0 ** -6, atol=2.0 ** -6)
    assert np.allclose(lse[:, 0::2], want_lse[:, 0::2], rtol=1e-5)
    assert np.isnan(out[:, 1::2]).all() and np.isnan(lse[:, 1::2]).all()
    _say("attention NaN score", new, kv, dim)
    p.kc[slot // 16, slot % 16, 0, 0] = float("nan")  # heads 0 and 1 read key head 0
    out, lse = p.run(gpu)
    assert np.isnan(out[:, :2]).all() and np.isnan(lse[:, :2]).all()
    assert np.allclose(out[:, 2], want[:, 2], rtol=2.0 ** -6, atol=2.0 ** -6)


@pytest.mark.parametrize("new", [1, 70])
def test_no_score_is_finite(gpu, new):
    _say("attention one key, not finite", new)
    for bad, want in ((float("nan"), np.nan), (float("-inf"), 0.0)):
        p = Problem("float16", [new], [new], 2, 1, 64, 16, seed=17)
        p.q[:, :, 0] = 1.0
        row = p.table[0].long()
        for j in range(new):
            p.kc[row[j // 16], j % 16, 0, 0] = bad
        out, lse = p.run(gpu)
        assert np.array_equal(out, np.full_like(out, want), equal_nan=True)
        assert np.array_equal(lse, np.full_like(lse, np.nan if want else -np.inf), equal_nan=True)


@pytest.mark.parametrize("hints", [{}, dict(max_new=1), dict(max_new=200)])
def test_arrays_that_make_no_sense_stay_inside(gpu, hints):
    """Offsets that do not ascend, lengths and slots out of range: answers of no meaning, inside the buffers."""
    import torch
    _say("attention with senseless arrays", hints)
    i32 = dict(dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(18)
    q = torch.randn(90, 4, 64, device="cuda").half()
    kc, vc = (torch.randn(600, 16, 2, 64, device="cuda").half() for _ in range(2))
    room = 512 * 16
    wild = lambda *s: torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, s).astype(np.int32)).cuda()  # noqa: E731
    for n in (5, 100):
        for starts in (torch.from_numpy(rng.integers(-40, 140, n + 1).astype(np.int32)).cuda(), wild(n + 1),
                       torch.arange(n, -1, -1, **i32)):
            for kv_len in (torch.full((n,), room, **i32), wild(n)):
                for selection in (None, (wild(n, room), kv_len, wild(90))):
                    table = torch.from_numpy(rng.integers(-5, 605, (n, 512)).astype(np.int32)).cuda()
                    wide = torch.full((94, 4, 64), 7.0, device="cuda").half()
                    lse = torch.full((94, 4), 7.0, device="cuda")
                    gpu.paged_attention(q, kc, vc, table, starts, kv_len, wide[2:92], d_lse=lse[2:92],
                                        selection=selection, **hints)
                    torch.cuda.synchronize()
                    for x in (wide, lse):
                        assert torch.all(x[:2] == 7.0) and torch.all(x[92:] == 7.0)


@pytest.mark.parametrize("density", [None, 0.4])
@pytest.mark.parametrize("what", [([256], [1500], 32, 4, 64, 16), ([100, 1, 90], [2100, 1800, 3], 33, 11, 96, 16),
                                  ([9] * 30, [4100] + [50] * 29, 16, 2, 192, 16)])
def test_many_rows_of_several_ranges(gpu, what, density):
    """More rows than are joined by a workgroup each, of requests with several ranges and with one."""
    _say("attention many rows joined", what, density)
    Problem("float16", *what, seed=19, density=density).check(gpu, max_new=max(what[0]), max_kv=max(what[1]))


@pytest.mark.parametrize("density", [None, 0.5])
@pytest.mark.parametrize("kv", [[4200, 70, 70, 40, 70], [4100] * 5, [70, 0, 70, 70, 4500]])
def test_tiles_of_uneven_requests(gpu, kv, density):
    """More than half of the card's places filled: cut only where the longest request stands out."""
    _say("attention uneven tiles", kv, density)
    p = Problem("bfloat16", [33] * 5, kv, 64, 64, 64, 16, seed=20, density=density)
    p.check(gpu, max_new=33)


@pytest.mark.parametrize("density", [None, 0.4])
@pytest.mark.parametrize("n", [63, 70, 128, 140])
def test_many_requests_of_single_tokens(gpu, n, density):
    """Requests without tokens or keys, of one key and of many, in any order of lengths."""
    _say("attention many requests", n, density)
    rng = np.random.default_rng(21)
    kv = (2 ** rng.uniform(0, 9, n)).astype(int)
    kv[::9], kv[5], kv[n - 1] = 0, 700, 511
    new = np.ones(n, int)
    new[3::11] = 0
    Problem("float16", new.tolist(), kv.tolist(), 4, 2, 64, 16, seed=22, density=density).check(gpu, max_new=1)


@pytest.mark.parametrize("density", [None, 0.5])
@pytest.mark.parametrize("new_of_the_longest", [0, 40])
@pytest.mark.parametrize("requests,heads", [(63, 8), (200, 2), (260, 1)])
def test_tiles_of_many_requests(gpu, requests, heads, new_of_the_longest, density):
    """More requests than a wave has lanes, in tiles for more than half of the card's places: the device cuts them where
    one stands out, and leaves them whole where the longest has no new tokens."""
    _say("attention tiles of many requests", requests, heads, new_of_the_longest, density)
    new, kv = [33 + i % 3 for i in range(requests)], [70 + i % 23 for i in range(requests)]
    p = Problem("bfloat16", new + [new_of_the_longest], kv + [4100], heads, heads, 64, 16, seed=23, density=density)
    p.check(gpu, max_new=40)


@pytest.mark.parametrize("below", [17.5, 19.0, 21.0])
@pytest.mark.parametrize("new,hints,sinks", [(1, dict(max_kv=100), [0, 32, 64, 96]), (40, dict(max_kv=200), [0])])
def test_many_small_probabilities_count_in_f16(gpu, new, hints, sinks, below):
    """A few keys that outdo 131072 others by e^17 and more, which together still weigh: each rounded probability is off by
    2^-11 of itself, or, below f16's normal range, by 2^-32 of the largest at most."""
    import torch
    _say("attention small probabilities", new, below)
    n = 131072
    p = Problem("float16", [new], [n], 1, 1, 64, 16, seed=24, causal=False)
    p.q[:], p.kc[:], p.vc[:] = 0, 0, 1
    p.q[:, :, 0] = 1.0
    for j in sinks:  # one for each wave that takes its own keys
        page = p.table[0, j // 16].long()
        p.kc[page, j % 16, 0, 0], p.vc[page, j % 16] = below, 0
    out, lse = p.run(gpu, scale=1.0, **hints)
    rest = (n - len(sinks)) * np.exp(-below)
    o0, z0 = rest / (len(sinks) + rest), below + np.log(len(sinks) + rest)
    ds = (64 + 8) * 2.0 ** -23 * below
    u = U["float16"]
    tol = 1.01 * (2 * u * o0 + n * 2.0 ** -32 + (2 * ds + n * 2.0 ** -24 + 2.0 ** -20) * o0)
    assert np.all(np.abs(out - o0) <= tol), (out.min(), out.max(), o0, tol)
    assert np.all(np.abs(lse - z0) <= ds + 2.0 ** -22 * (z0 + np.log(n) + 2) + n * 2.0 ** -24)
    assert torch.isfinite(p.vc).all()


def test_strides_of_axes_of_one_entry(gpu):
    """One token, one key head, one page, a table of one row: their strides lead nowhere, and may be odd numbers."""
    import torch
    _say("attention odd strides of single entries")
    p = Problem("float16", [1], [11], 3, 1, 64, 16, seed=25)
    row, one = p.table[0, :1].clone(), dict(scale=0.125, max_new=1)
    kc, vc = (x[row.long()].clone() for x in (p.kc, p.vc))
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    want, got = torch.zeros_like(p.q), torch.zeros(1, 3, 64, device="cuda").half()
    gpu.paged_attention(p.q, kc, vc, table, p.starts, p.kv_len, want, **one)
    odd = lambda x, *stride: torch.as_strided(x, x.shape, stride)  # noqa: E731
    gpu.paged_attention(odd(p.q, 1, 64, 1), odd(kc, 3, 64, 1, 1), odd(vc, 5, 64, 7, 1), odd(table, 0, 1), p.starts,
                        p.kv_len, odd(got, 1, 64, 1), **one)
    torch.cuda.synchronize()
    assert torch.equal(want, got) and torch.isfinite(got).all() and got.abs().sum() > 0
    # with one slot a page, its stride leads nowhere either
    kc, vc = (x[:, :1].clone() for x in (kc, vc))
    gpu.paged_attention(p.q, kc, vc, table, p.starts, torch.ones_like(p.kv_len), want, **one)
    gpu.paged_attention(p.q, odd(kc, 3, 9, 1, 1), odd(vc, 1, 1, 1, 1), table, p.starts, torch.ones_like(p.kv_len), got, **one)
    torch.cuda.synchronize()
    assert torch.equal(want, got)
