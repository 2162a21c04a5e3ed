"""paged_weights against the formula in 64 bits.

The bar of a weight, the sum of terms p = e^(s - lse): a score is an fp32 sum of
exact products, off by (dim + 8) 2^-23 |scale| sum|q k|; its scale, the log-sum and
their difference are each rounded once in powers of two (2^-24 of |s|, |lse| and
|s - lse|), the exponential to 2^-22 of itself; n terms are summed in fp32 (n 2^-24
of the sum); what was there before is rounded twice.
"""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


class Problem:
    """Requests over a paged cache, the pages scattered and what nobody sees full of NaN; lse is as an attention over
    all that a row sees leaves it, or any."""

    def __init__(self, dtype, new, kv, heads, kv_heads, dim, page, seed=0, spread=2.0, layout="plain", density=None,
                 causal=True, scale=None, lse=None, extra=0):
        import torch
        self.torch, self.dtype, self.page, self.causal = torch, dtype, page, causal
        self.new, self.kv, self.heads, self.kv_heads, self.dim = list(new), list(kv), heads, kv_heads, dim
        self.scale = dim ** -0.5 if scale is None else scale
        dt = getattr(torch, dtype)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        held = [-(-max(0, x) // page) for x in kv]
        self.cols = max(1, max(held, default=1))
        self.pages = sum(held) + 3
        order = torch.randperm(self.pages, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(kv), self.cols + 2), -1, dtype=torch.int32, device="cuda")[:, :self.cols]
        at = 0
        for r, n in enumerate(held):
            self.table[r, :n] = order[at:at + n]
            at += n
        if layout == "heads first":
            self.kc = rnd(self.pages, kv_heads, page, dim).to(dt).transpose(1, 2)
        elif layout == "padded":
            self.kc = rnd(self.pages, page, kv_heads, dim + 16).to(dt)[..., 8:8 + dim]
        else:
            self.kc = rnd(self.pages, page, kv_heads, dim).to(dt)
        self.kc[order[at:].long()] = float("nan")
        for r, n in enumerate(held):
            if n and kv[r] % page:
                self.kc[self.table[r, n - 1].long(), kv[r] % page:] = float("nan")
        total = sum(new) + extra  # rows behind the last request's are not looked at
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
            self.visible = torch.rand(self.pages * page, device="cuda", generator=g) < density
            self.kc[~self.visible.view(self.pages, page)] = float("nan")
        self.past = 5 * torch.rand(len(kv), self.cols * page + 3, device="cuda", generator=g)
        self.lse = torch.zeros(total, heads, device="cuda") if lse is None else torch.full((total, heads), lse, device="cuda")
        if lse is None:
            for r, row, see, s, _ in self.rows():
                z = np.log(np.exp(s - s.max()).sum()) + s.max() if len(s) else -np.inf
                self.lse[row] = float(z)

    def rows(self):
        """(request, (token, head), the positions that it sees, their scores, the size of the scores' terms)."""
        host = lambda t: t.double().cpu().numpy()  # noqa: E731
        q, kc, table = host(self.q), host(self.kc), self.table.cpu().numpy()
        visible = None if self.visible is None else self.visible.cpu().numpy()
        group, at = self.heads // self.kv_heads, 0
        for r, (n, kv) in enumerate(zip(self.new, self.kv)):
            pos = np.arange(max(0, kv))
            page, off = table[r, pos // self.page], pos % self.page
            there = (page >= 0) & (page < self.pages)
            if visible is not None:
                there &= visible[np.where(there, page, 0) * self.page + off]
            for i in range(n):
                see = pos[there & ((pos <= kv - n + i) if self.causal else True)]
                for h in range(self.heads):
                    k = kc[page[see], off[see], h // group]
                    yield (r, (at + i, h), see, self.scale * (k @ q[at + i, h]),
                           abs(self.scale) * (np.abs(k) @ np.abs(q[at + i, h])))
            at += n

    def run(self, gpu, past=True, decay=0.75, kind="bitmap", in_place=False, **kw):
        torch = self.torch
        out = torch.full((len(self.kv), self.cols * self.page + 5), 7.0, device="cuda")
        if in_place:
            out[:, :self.past.shape[1]] = self.past
        g = None
        if self.visible is not None:
            ids = np.nonzero(self.visible.cpu().numpy())[0].astype(np.uint32)
            g = gpu.upload_from_ids(ids, self.visible.numel(),
                                    gpu.PROMOTE_ALL if kind == "bitmap" else gpu.PROMOTE_KEEP_DEFAULT)
        gpu.paged_weights(self.q, self.kc, self.table, kw.pop("starts", self.starts), kw.pop("kv_len", self.kv_len),
                          self.lse, out, d_past=(out if in_place else self.past) if past else None, decay=decay,
                          scale=self.scale, causal=self.causal, visible=g, **kw)
        torch.cuda.synchronize()
        if g is not None:
            gpu.free(g)
        return out.cpu().numpy().astype(np.float64)

    def check(self, gpu, past=True, decay=0.75, out=None, **kw):
        out = self.run(gpu, past, decay, **kw) if out is None else out
        before = self.past.cpu().numpy().astype(np.float64)
        want, tol = np.zeros(out.shape), np.zeros(out.shape)
        terms = np.zeros(len(self.kv))
        lse = self.lse.cpu().numpy().astype(np.float64)
        for r, row, see, s, size in self.rows():
            z = lse[row]
            terms[r] += 1
            if z == -np.inf:
                continue
            p = np.exp(s - z)
            ds = (self.dim + 8) * 2.0 ** -23 * size
            want[r, see] += p
            tol[r, see] += p * (ds + 2.0 ** -24 * (2 * np.abs(s) + np.abs(z) + np.abs(s - z)) + 2.0 ** -22)
        for r, (n, kv) in enumerate(zip(self.new, self.kv)):
            kv = max(0, kv)
            tol[r] += (terms[r] + 4) * 2.0 ** -24 * want[r]
            if past:
                old = max(0, self.kv[r] - n)
                want[r, :old] += np.float32(decay) * before[r, :old]
                tol[r, :old] += 2.0 ** -22 * before[r, :old]
            if kw.get("in_place"):
                assert np.array_equal(out[r, kv:self.past.shape[1]], before[r, kv:])
            else:
                assert np.all(out[r, kv:] == 7.0), "entries behind the request's last"
            bad = np.abs(out[r, :kv] - want[r, :kv]) > 1.01 * tol[r, :kv]
            assert not bad.any(), (r, np.nonzero(bad)[0][:5], out[r, :kv][bad][:5], want[r, :kv][bad][:5])


# new, kv, heads, key heads, dim, page
SHAPES = {
    "one token, one key": ([1], [1], 1, 1, 64, 16),
    "short context": ([1], [37], 8, 2, 128, 16),
    "decode ragged": ([1, 1, 1, 1, 1], [1, 16, 17, 300, 1025], 8, 2, 128, 16),
    "decode mha": ([1, 1, 1], [63, 64, 65], 5, 5, 64, 32),
    "decode wide group": ([1, 1], [200, 129], 24, 1, 128, 8),
    "decode group 33": ([1], [150], 33, 1, 64, 16),
    "three key heads": ([1, 2], [150, 70], 6, 3, 64, 16),
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
def test_weights(gpu, dtype, what):
    _say("weights", dtype, what)
    p = Problem(dtype, *SHAPES[what], seed=len(what), extra=2)
    p.check(gpu)
    p.check(gpu, past=False)


@pytest.mark.parametrize("kind", ["bitmap", "arrays"])
@pytest.mark.parametrize("density", [0.0, 0.02, 0.4, 1.0])
@pytest.mark.parametrize("what", ["decode ragged", "a few tokens", "chunk", "prompt group 3", "pages of one"])
def test_weights_of_what_a_filter_lets_through(gpu, what, density, kind):
    _say("weights filtered", what, density, kind)
    Problem("float16", *SHAPES[what], seed=3, density=density).check(gpu, kind=kind)


@pytest.mark.parametrize("what", ["decode ragged", "chunk", "more tokens than positions"])
def test_weights_not_causal(gpu, what):
    _say("weights not causal", what)
    Problem("bfloat16", *SHAPES[what], seed=4, causal=False).check(gpu)


@pytest.mark.parametrize("layout", ["heads first", "padded"])
@pytest.mark.parametrize("what", ["decode ragged", "chunk", "dims 80"])
def test_weights_strides(gpu, what, layout):
    _say("weights strides", what, layout)
    Problem("bfloat16", *SHAPES[what], seed=5, layout=layout).check(gpu, in_place=True)


@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 1.0), (0.3, 8.0), (1e-3, 1.0)])
@pytest.mark.parametrize("what", ["decode ragged", "chunk"])
def test_weights_scales(gpu, what, scale, spread):
    _say("weights scale", what, scale)
    Problem("float16", *SHAPES[what], seed=6, spread=spread, scale=scale).check(gpu)


@pytest.mark.parametrize("hints", [dict(max_new=1, max_kv=1), dict(max_new=5000, max_kv=1 << 20), dict(max_kv=200),
                                   dict(max_new=2)])
@pytest.mark.parametrize("what", ["decode ragged", "chunk", "three key heads"])
def test_hints_do_not_change_the_answer(gpu, what, hints):
    _say("weights hints", what, hints)
    Problem("bfloat16", *SHAPES[what], seed=7).check(gpu, **hints)


@pytest.mark.parametrize("max_new", [1, 5000])
@pytest.mark.parametrize("what", SHAPES)
def test_either_way_of_splitting(gpu, what, max_new):
    """Every shape by the kernel for few rows and by the one for many."""
    _say("weights either way", what, max_new)
    Problem("float16", *SHAPES[what], seed=21, density=0.7, extra=1).check(gpu, max_new=max_new)


@pytest.mark.parametrize("new,kv", [([1], [20011]), ([1, 1], [5000, 12345]), ([17], [9000]), ([33, 2], [6000, 40])])
def test_weights_long_contexts(gpu, new, kv):
    _say("weights long", new, kv)
    Problem("bfloat16", new, kv, 8, 2, 128, 16, seed=8).check(gpu)
    Problem("float16", new, kv, 4, 4, 64, 32, seed=9, density=0.2).check(gpu)


def test_a_prompt_of_many_rows(gpu):
    _say("weights of many rows")
    Problem("bfloat16", [700], [900], 8, 2, 64, 16, seed=18).check(gpu)


@pytest.mark.parametrize("what", [([700, 5, 90], [900, 300, 400], 8, 2, 64, 16), ([3, 400, 0, 100], [800, 400, 20, 100], 8, 2, 128, 16),
                                  ([600, 80], [600, 2000], 4, 1, 256, 16)])
def test_uneven_requests_after_others(gpu, what):
    """Requests with fewer parts of rows than the longest, in a workspace that another call has left its sums in."""
    _say("weights of uneven requests", what[0])
    for density in (None, 0.5):
        p = Problem("bfloat16", *what, seed=22, density=density)
        lse = p.lse
        for more in (40.0, float("nan")):
            p.lse = lse - more
            p.run(gpu)
            p.lse = lse
            p.check(gpu)


@pytest.mark.parametrize("density", [None, 0.4])
@pytest.mark.parametrize("hint", ["none", "longest", "short"])
@pytest.mark.parametrize("what", [([300] + [1] * 20, [600] + [90] * 20, 8, 2, 64, 16), ([1] * 9 + [80, 1, 40, 0], [130] * 13, 8, 2, 128, 16),
                                  ([1] * 1030 + [120, 1], [20] * 1030 + [150, 40], 2, 1, 64, 16), ([1, 1, 60, 1, 1], [700] * 5, 4, 1, 256, 16),
                                  ([2] * 6 + [200] * 2, [300] * 8, 3, 1, 80, 16)])
def test_long_requests_among_short_ones(gpu, what, hint, density):
    _say("weights of long and short", what[0][:3], len(what[0]), hint, density)
    p = Problem("bfloat16", *what, seed=24, density=density, extra=1)
    p.check(gpu, max_new={"none": 0, "longest": max(what[0]), "short": 60}[hint])


def test_a_captured_call_goes_by_the_lengths_it_finds(gpu):
    """Replays after another request has become the long one."""
    import torch
    _say("weights captured, other lengths")
    news = [[120] + [1] * 12, [1] * 12 + [120], [1, 60, 1, 1, 61] + [1] * 8, [7] * 8 + [15, 14, 16, 16, 15], [0] * 12 + [132]]
    p = Problem("bfloat16", news[0], [150] * 13, 8, 2, 64, 16, seed=26)
    q, lse, out = p.q, p.lse, torch.zeros(13, p.cols * 16, device="cuda")
    call = lambda s: gpu.paged_weights(q, p.kc, p.table, p.starts, p.kv_len, lse, out, max_new=132, max_kv=150, stream=s)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(side)
    for new in news + news[:2]:
        starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        with torch.cuda.stream(side):
            p.starts.copy_(starts)
            call(side)
            want = out.clone()
            out.zero_()
            graph.replay()
        side.synchronize()
        assert torch.equal(out, want) and bool(want.abs().sum() > 0), new
        p.new, p.q, p.lse = new, q, lse
        got = np.full((13, p.cols * 16 + 5), 7.0)
        got[:, :150] = out.cpu().numpy()[:, :150]
        p.check(gpu, past=False, out=got)


def test_many_long_requests_of_the_same_rows(gpu):
    """More rows in all than there are: what a list has no room for is answered all the same."""
    import torch
    _say("weights of shared rows, uneven")
    i32 = dict(dtype=torch.int32, device="cuda")
    n = 60
    p = Problem("bfloat16", [90] + [0] * (n - 1), [200] * n, 4, 1, 64, 16, seed=25)
    starts = [0, 90] * (n // 2) + [0]  # every second request counts all rows, the ones between none
    got = p.run(gpu, starts=torch.tensor(starts, **i32), max_new=90)
    p.new = [max(0, b - a) for a, b in zip(starts, starts[1:])]
    p.q, p.lse = torch.cat([p.q[:90]] * (n // 2)), torch.cat([p.lse[:90]] * (n // 2))
    p.check(gpu, out=got)


def test_rows_that_count_for_nothing(gpu):
    """Rows whose log-sum is -inf, as those that saw nothing leave it."""
    _say("weights of rows that saw nothing")
    p = Problem("bfloat16", [3, 40], [50, 60], 4, 2, 64, 16, seed=10, lse=float("-inf"))
    out = p.run(gpu, past=False)
    assert np.all(out[0, :50] == 0) and np.all(out[1, :60] == 0)
    p.lse[1:3] = 2.0
    p.check(gpu)


@pytest.mark.parametrize("what", ["decode ragged", "a few tokens", "chunk", "prompt", "dims 192", "dims 256"])
def test_rows_that_count_for_nothing_may_hold_anything(gpu, what):
    """Padding: queries that are NaN or infinite, with a log-sum of -inf."""
    _say("weights of rows that hold anything", what)
    p = Problem("bfloat16", *SHAPES[what], seed=20)
    gone = [(t, h) for t in range(0, p.q.shape[0], 3) for h in range(t % 2, p.heads, 2)]
    for t, h in gone:
        p.lse[t, h] = float("-inf")
    want = p.run(gpu)
    for i, (t, h) in enumerate(gone):
        p.q[t, h] = float("nan") if i % 2 else float("inf")
    assert np.array_equal(p.run(gpu), want)


def test_weights_add_up_to_the_rows(gpu):
    """A row's weights sum to one: the attention's own log-sum goes in, and out comes the number of rows."""
    import torch
    _say("weights after the attention")
    for new, kv, heads, kv_heads, dim in (([1, 1], [700, 33], 8, 2, 128), ([64, 20], [300, 20], 6, 2, 64)):
        p = Problem("bfloat16", new, kv, heads, kv_heads, dim, 16, seed=11)
        out = torch.empty_like(p.q)
        gpu.paged_attention(p.q, p.kc, p.kc, p.table, p.starts, p.kv_len, out, d_lse=p.lse)
        w = p.run(gpu, past=False)
        for r, (n, m) in enumerate(zip(new, kv)):
            assert abs(w[r, :m].sum() - n * heads) < 1e-4 * n * heads  # scores of +-30 in fp32: some 2^-17 of a weight


def test_some_rows_of_a_request(gpu):
    """The last tokens of a prompt, and the first of a verified draft, as d_new says."""
    import torch
    _say("weights of some rows")
    i32 = dict(dtype=torch.int32, device="cuda")
    p = Problem("float16", [40, 7, 5], [90, 60, 5], 4, 2, 64, 16, seed=12)
    whole = Problem("float16", [40, 7, 5], [90, 60, 5], 4, 2, 64, 16, seed=12)
    # the last 8 tokens of each (all, where there are fewer)
    take = [8, 7, 5]
    starts = torch.tensor([32, 40, 47], **i32)
    got = p.run(gpu, starts=starts, d_new=torch.tensor(take, **i32))
    p.new, p.q, p.lse = take, torch.cat([p.q[32:40], p.q[40:47], p.q[47:52]]), torch.cat([p.lse[32:40], p.lse[40:]])
    p.starts = torch.tensor([0, 8, 15, 20], **i32)
    p.check(gpu, out=got)
    p.check(gpu)
    # the first 3, 0 and 5 tokens, the requests cut off behind them
    p, take, kv = whole, [3, 0, 5], [53, 53, 5]
    got = p.run(gpu, starts=p.starts, kv_len=torch.tensor(kv, **i32), d_new=torch.tensor(take, **i32))
    p.q, p.lse = torch.cat([p.q[:3], p.q[47:52]]), torch.cat([p.lse[:3], p.lse[47:52]])
    p.new, p.kv, p.kv_len, p.starts = take, kv, torch.tensor(kv, **i32), torch.tensor([0, 3, 3, 8], **i32)
    p.check(gpu, out=got)
    p.check(gpu)


def test_rows_of_several_requests(gpu):
    """Requests that count the same rows, more of them in all than there are, and in any order."""
    import torch
    _say("weights of shared rows")
    i32 = dict(dtype=torch.int32, device="cuda")
    n, take = 40, 70
    p = Problem("bfloat16", [take + 30] + [0] * (n - 1), [500] * n, 4, 1, 64, 16, seed=19)
    starts = [(7 * i) % 31 for i in range(n)]
    got = p.run(gpu, starts=torch.tensor(starts, **i32), d_new=torch.full((n,), take, **i32))
    p.new, p.q = [take] * n, torch.cat([p.q[s:s + take] for s in starts])
    p.lse = torch.cat([p.lse[s:s + take] for s in starts])
    p.check(gpu, out=got)


def test_pages_outside_the_cache_get_nothing(gpu):
    _say("weights with pages outside the cache")
    p = Problem("bfloat16", [1, 40], [100, 90], 4, 2, 64, 16, seed=13)
    p.table[0, 2], p.table[1, 1] = -1, p.pages
    out = p.run(gpu, past=False)
    assert np.all(out[0, 32:48] == 0) and np.all(out[1, 16:32] == 0)
    p.check(gpu)


def test_senseless_device_data_stays_inside(gpu):
    import torch
    _say("weights of noise")
    p = Problem("bfloat16", [3, 2, 4], [50, 40, 30], 4, 2, 64, 16, seed=14)
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(20):
        noise = lambda n: torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=g, device="cuda").to(torch.int32)  # noqa: E731
        p.starts, p.kv_len = noise(4), noise(3)
        p.table = noise(3 * p.cols).view(3, p.cols)
        d_new = noise(3) if i % 2 else None
        out = p.run(gpu, d_new=d_new)
        assert np.all(out[:, p.cols * 16:] == 7.0)


def test_two_runs_give_the_same_bits(gpu):
    _say("weights twice")
    for what in ("decode ragged", "chunk", "a few tokens", "prompt"):
        p = Problem("bfloat16", *SHAPES[what], seed=15)
        assert np.array_equal(p.run(gpu), p.run(gpu))


def test_another_stream(gpu):
    import torch
    _say("weights on another stream")
    p = Problem("bfloat16", *SHAPES["chunk"], seed=16)
    want = p.run(gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = p.run(gpu, stream=s)
    assert np.array_equal(got, want)


def test_offsets_past_32_bits(gpu):
    """A cache whose keys lie more than 2^32 elements apart."""
    import torch
    _say("weights past 32 bits")
    pages, page, dim = 300, 16, 64
    held = torch.empty(5 * 2 ** 30, dtype=torch.bfloat16, device="cuda")
    step = (held.numel() - page * dim) // (pages - 1) // 8 * 8
    kc = held.as_strided((pages, page, 1, dim), (step, dim, dim, 1))
    p = Problem("bfloat16", [1], [pages * page - 50], 2, 1, dim, page, seed=17)
    kc.copy_(p.kc[:pages])
    p.table.clamp_(max=pages - 1)
    want = p.run(gpu)
    p.kc = kc
    assert np.array_equal(p.run(gpu), want, equal_nan=True)
