"""The operators for long and speculative answers where their arguments meet: sets that are narrower than what they are
asked about, and rows that count for nothing beside keys that hold anything."""
import numpy as np
import pytest

import test_gpu_evict
import test_gpu_verify
import test_gpu_weights

pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


class Narrow(test_gpu_verify.Problem):
    """Allowed tokens as a bitmap whose universe ends before the scores do."""

    def __init__(self, universe, *args, **kw):
        super().__init__(*args, **kw)
        self.universe = universe
        self.allowed[:, universe:] = False

    def run(self, gpu, most=None, stream=None):
        import torch
        ids = np.nonzero(self.allowed[0])[0].astype(np.uint32)
        allowed = gpu.upload_from_ids(ids, self.universe, gpu.PROMOTE_ALL)
        assert allowed.negated and allowed.n_bitmap_containers == allowed.n_containers
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        i32, n = dict(dtype=torch.int32, device="cuda"), len(self.rows)
        starts = cuda(np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32))
        accepted, out = torch.full((n,), -9, **i32), torch.full((n, max(self.rows)), -9, **i32)
        gpu.draft_verify(self.x, cuda(self.tokens), starts, cuda(self.uniform), accepted, out, d_draft=self.draft,
                         temperature=self.temperature, allowed=allowed)
        torch.cuda.synchronize()
        gpu.free(allowed)
        return accepted.cpu().numpy(), out.cpu().numpy()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows", [[4, 3, 5], [14, 20]])
@pytest.mark.parametrize("universe,vocab", [(1000, 1100), (65536, 65700), (70000, 70400), (70016, 140000), (3000, 70000)])
def test_drafts_behind_the_universe(gpu, universe, vocab, rows, draft):
    """Tokens that scores have room for and the set of allowed ones says nothing of, the model's favourites among them."""
    _say("verify behind the universe", universe, vocab, rows, draft)
    p = Narrow(universe, rows, vocab, "bfloat16", seed=31, density=0.9, kind="bitmap", draft=draft)
    for i in range(1, len(p.tokens), 2):
        d = int(p.rng.integers(universe, vocab))
        p.tokens[i] = d
        p.x[i - 1, d] = 30.0
    p.check(gpu)


@pytest.mark.parametrize("kind", ["bitmap", "arrays"])
@pytest.mark.parametrize("positions", [True, False])
def test_pinned_slots_of_the_first_pages_alone(gpu, kind, positions):
    """A bitmap of pinned slots that knows only the first pages says nothing of the others: their tokens move."""
    import torch
    _say("evict, few pinned pages", kind, positions)
    page, n_pages, kv, keep = 16, 40, 600, 250
    rng = np.random.default_rng(32)
    i32 = dict(dtype=torch.int32, device="cuda")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    table = rng.permutation(n_pages).astype(np.int32)[None, :38]
    w = rng.random((1, 38 * page)).astype(np.float32)
    at = rng.permutation(38 * page).astype(np.int32)[None]
    pinned = np.zeros(n_pages * page, bool)
    pinned[:5 * page] = rng.random(5 * page) < (0.8 if kind == "bitmap" else 0.3)
    g = gpu.upload_from_ids(np.nonzero(pinned)[0].astype(np.uint32), 5 * page,
                            gpu.PROMOTE_ALL if kind == "bitmap" else gpu.PROMOTE_KEEP_DEFAULT)
    one = lambda x: torch.tensor([x], **i32)  # noqa: E731
    out, p_out, length, n_moves = torch.zeros(1, 38 * page, device="cuda"), torch.zeros(1, 38 * page, **i32), one(-9), one(-9)
    moves, freed, counts = torch.full((1, 19 * page, 2), -9, **i32), torch.full((38,), -9, **i32), torch.zeros(2, **i32)
    gpu.paged_evict(cuda(w), one(kv), one(keep), cuda(table), page, out, length, moves, n_moves, freed, counts,
                    d_positions=cuda(at) if positions else None, d_kept=one(kv) if positions else None,
                    d_seen=one(kv) if positions else None, d_positions_out=p_out, sinks=2, recent=4, pinned=g)
    torch.cuda.synchronize()
    gpu.free(g)
    m, lies, pos, want, cols = test_gpu_evict.evict_oracle(w[0], at[0], kv if positions else 0, kv, kv, keep, table[0], page,
                                                           n_pages, 2, 4, pinned)
    assert int(length[0]) == m and int(n_moves[0]) == len(want) > 0
    assert moves[0, :len(want)].tolist() == [list(x) for x in want]
    assert np.array_equal(out[0, :m].cpu().numpy(), w[0][lies]) and p_out[0, :m].tolist() == [pos[i] for i in lies]


@pytest.mark.filterwarnings("ignore:invalid value encountered")
@pytest.mark.parametrize("density", [None, 0.8])
@pytest.mark.parametrize("max_new", [1, 5000])
@pytest.mark.parametrize("what", ["a few tokens", "chunk", "prompt group 3", "dims 192", "dims 256"])
def test_rows_that_count_for_nothing_beside_any_keys(gpu, what, max_new, density):
    """Positions that only rows with a log-sum of -inf see, whose keys are NaN or infinite, got nothing."""
    _say("weights, any keys", what, max_new, density)
    p = test_gpu_weights.Problem("bfloat16", *test_gpu_weights.SHAPES[what], seed=33, density=density)
    at = 0
    for r, (n, kv) in enumerate(zip(p.new, p.kv)):
        gone = min(n, 3)
        for i in range(gone):
            p.lse[at + n - 1 - i] = float("-inf")
            position = kv - 1 - i
            p.kc[p.table[r, position // p.page].long(), position % p.page] = float("nan") if i % 2 else float("inf")
        at += n
    out = p.run(gpu, max_new=max_new)
    for r, kv in enumerate(p.kv):
        assert np.isfinite(out[r, :kv]).all(), (r, np.nonzero(~np.isfinite(out[r, :kv]))[0])
    p.check(gpu, out=out)


@pytest.mark.parametrize("density", [None, 0.4])
@pytest.mark.parametrize("max_new", [1, 5000])
@pytest.mark.parametrize("what", test_gpu_weights.SHAPES)
def test_weights_are_finite(gpu, what, max_new, density):
    """Keys that nobody sees are NaN in all of these: a comparison of differences alone would let theirs pass."""
    _say("weights finite", what, max_new, density)
    p = test_gpu_weights.Problem("bfloat16", *test_gpu_weights.SHAPES[what], seed=36, density=density)
    out = p.run(gpu, max_new=max_new)
    assert all(np.isfinite(out[r, :max(0, kv)]).all() for r, kv in enumerate(p.kv))
    p.check(gpu, out=out)


def _requests(gpu, n, cols, heads, kv_heads, hints, tokens=1, seed=37):
    """Weights of n short requests in rows of `cols` pages of 16, by calls of the given numbers of requests."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    i32, dim, pages = dict(dtype=torch.int32, device="cuda"), 8, 512
    table = torch.full((n, cols), -1, **i32)
    table[:, :2] = torch.randint(0, pages, (n, 2), device="cuda", generator=g).to(torch.int32)
    kc = torch.randn(pages, 16, kv_heads, dim, device="cuda", generator=g).half()
    q = torch.empty(n * tokens, heads, dim, device="cuda", dtype=torch.float16).normal_(generator=g)
    lse = torch.full((n * tokens, heads), 3.0, device="cuda")
    kv_len = torch.randint(1, 33, (n,), device="cuda", generator=g).to(torch.int32)
    starts = torch.arange(0, n * tokens + 1, tokens, **i32)

    def weights(each):
        out = torch.full((n, cols * 16), 7.0, device="cuda")
        for r in range(0, n, each):
            s = slice(r, r + each)
            gpu.paged_weights(q[r * tokens:(r + each) * tokens], kc, table[s], starts[r:r + each + 1] - starts[r], kv_len[s],
                              lse[r * tokens:(r + each) * tokens], out[s], **hints)
        torch.cuda.synchronize()
        return out, kv_len

    return weights


def test_more_requests_than_a_launch_holds(gpu):
    """131072 requests of 65 rows to each of 64 key heads: 2^23 workgroups."""
    import torch
    _say("weights, more than a launch")
    weights = _requests(gpu, 1 << 17, 2, 64 * 65, 64, dict(max_new=1))
    got, kv_len = weights(1 << 17)
    want, _ = weights(1 << 15)
    seen = torch.arange(32, device="cuda")[None] < kv_len[:, None]
    assert torch.equal(got, want) and bool((got[seen] > 0).all()) and bool((got[~seen] == 7.0).all())


@pytest.mark.parametrize("hints", [{}, dict(max_kv=1 << 17, max_new=1), dict(max_kv=32)])
def test_many_requests_in_wide_tables(gpu, hints):
    """4096 single tokens whose tables have room for 131072 positions each: refused with no launch of that size to make."""
    import torch
    _say("weights in wide tables", hints)
    got, kv_len = _requests(gpu, 4096, 8192, 16, 8, hints)(4096)
    want, _ = _requests(gpu, 4096, 2, 16, 8, {})(4096)
    assert torch.equal(got[:, :32], want) and bool((got[:, 32:] == 7.0).all())
    assert bool((want[:, 0] > 0).all())


@pytest.mark.parametrize("max_new", [0, 40, 20])
@pytest.mark.parametrize("some", [False, True])
def test_the_last_tokens_of_a_prompt(gpu, some, max_new):
    """Starts moved up to the tokens that count, in a q that holds all of them; a hint that is too small changes nothing."""
    import torch
    _say("weights of a prompt's last tokens", some, max_new)
    i32 = dict(dtype=torch.int32, device="cuda")
    p = test_gpu_weights.Problem("bfloat16", [700], [900], 8, 2, 128, 16, seed=38)
    if some:
        got = p.run(gpu, starts=torch.tensor([660], **i32), d_new=torch.tensor([40], **i32), max_new=max_new)
    else:
        got = p.run(gpu, starts=torch.tensor([660, 700], **i32), max_new=max_new)
    p.new, p.q, p.lse = [40], p.q[660:].contiguous(), p.lse[660:].contiguous()
    p.check(gpu, out=got)


@pytest.mark.parametrize("what", [
    # tokens of each request, heads, key heads, room: sums of some requests or some parts of rows at a time
    ([64] * 300, 32, 8, 65536), ([10000], 32, 8, 1 << 20), ([9000, 100, 0, 12000], 32, 8, 1 << 20),
    ([1] * 450 + [10000] + [1] * 400 + [70] + [1] * 48, 256, 64, 131072)])
def test_sums_that_do_not_fit_at_once(gpu, what):
    """The same requests in tables of just their positions and in wide ones, whose sums go launch after launch.  Either
    adds the same n terms in an order of its own, n 2^-24 of the sum off at most, and may multiply by the other kernel:
    a score is (dim + 8) 2^-23 of the size of its terms off, its difference to the log-sum 2^-24 of each, the exponential
    2^-22."""
    import torch
    tokens, heads, kv_heads, room = what
    _say("weights whose sums do not fit", len(tokens), max(tokens), room)
    g = torch.Generator(device="cuda").manual_seed(39)
    i32, dim, n, total = dict(dtype=torch.int32, device="cuda"), 64, len(tokens), sum(tokens)
    most = max(t + 300 for t in tokens)
    cols, pages = -(-most // 16), 1024
    near = torch.randint(0, pages, (n, cols), device="cuda", generator=g).to(torch.int32)
    wide = torch.full((n, room // 16), -1, **i32)
    wide[:, :cols] = near
    kc = torch.randn(pages, 16, kv_heads, dim, device="cuda", generator=g).half()
    q = torch.empty(total, heads, dim, device="cuda", dtype=torch.float16).normal_(generator=g)
    lse = torch.rand(total, heads, device="cuda", generator=g) + 8
    starts = torch.tensor(np.concatenate([[0], np.cumsum(tokens)]).astype(np.int32)).cuda()
    kv_len = torch.tensor([t + 7 * r % 300 for r, t in enumerate(tokens)], **i32)
    outs = []
    for table in (near, wide):
        out = torch.full((n, table.shape[1] * 16), 7.0, device="cuda")
        out[:, :cols * 16] = 0.25
        gpu.paged_weights(q, kc, table, starts, kv_len, lse, out, d_past=out, decay=0.5)
        outs.append(out[:, :cols * 16])
        assert bool((out[:, cols * 16:] == 7.0).all())
    torch.cuda.synchronize()
    rows = torch.tensor(tokens, device="cuda")[:, None] * (heads // kv_heads) * kv_heads
    seen = torch.arange(cols * 16, device="cuda")[None] < kv_len[:, None]
    near, wide = outs
    assert bool((near[seen] > 0).all()) and bool((near[~seen] == 0.25).all()) and bool((wide[~seen] == 0.25).all())
    size = dim ** -0.5 * float(q.float().norm(dim=-1).max()) * float(kc.float().norm(dim=-1).max())  # of a score's terms
    off = (dim + 8) * 2.0 ** -23 * size + 2.0 ** -24 * (3 * size + 2 * 9) + 2.0 ** -22
    terms = (rows / 16 + 64).expand_as(near)  # (a lane adds sixteen rows in pairs, so that no chain is longer)
    assert bool(((near - wide).abs() <= 2 * (off + terms * 2.0 ** -24) * near).all()), ((near - wide).abs() / near).max()


def _layers(n, seed=35):
    """The weights of n layers, whose rows are many: (call(i, out, stream), the calls' own results)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    requests, tokens, heads, kv_heads, dim, page, cols = 16, 64, 32, 8, 64, 16, 4096
    i32 = dict(dtype=torch.int32, device="cuda")
    half = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    table = torch.arange(requests * 4, **i32).view(requests, 4).repeat(1, cols // 4)
    kc = half(requests * 4, page, kv_heads, dim)
    q = [half(requests * tokens, heads, dim) for _ in range(n)]
    starts, kv_len = torch.arange(0, requests * tokens + 1, tokens, **i32), torch.full((requests,), tokens, **i32)
    lse = torch.full((requests * tokens, heads), 4.0, device="cuda")

    def call(gpu, i, out, stream):
        gpu.paged_weights(q[i], kc, table, starts, kv_len, lse, out, max_new=tokens, stream=stream)

    return call, lambda: torch.zeros(requests, cols * page, device="cuda")


def test_captured_layers_share_their_workspace(gpu):
    """The calls of one capture on one stream follow one another: their workspaces, 32 MB each, are one block.  Replays
    give what eager calls give."""
    import torch
    _say("captured layers")
    n = 24
    call, room = _layers(n)
    outs = [room() for _ in range(n)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(n):
            call(gpu, i, outs[i], side)
    side.synchronize()
    wants = [t.clone() for t in outs]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    with torch.cuda.graph(graph, stream=side):
        for i in range(n):
            call(gpu, i, outs[i], side)
    torch.cuda.synchronize()
    taken = free - torch.cuda.mem_get_info()[0]
    assert taken < 4 * 32 << 20, taken
    for _ in range(3):
        with torch.cuda.stream(side):
            for t in outs:
                t.zero_()
            graph.replay()
            call(gpu, 0, room(), side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))


def test_captured_streams_do_not_share(gpu):
    """Calls on two streams of one capture run side by side, each in a workspace of its own, as do two graphs."""
    import torch
    _say("captured streams")
    call, room = _layers(4)
    outs = [room() for _ in range(4)]
    for i in range(4):
        call(gpu, i, outs[i], None)
    torch.cuda.synchronize()
    wants = [t.clone() for t in outs]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for first in (0, 2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=one):
            two.wait_stream(one)
            call(gpu, first, outs[first], one)
            with torch.cuda.stream(two):
                call(gpu, first + 1, outs[first + 1], two)
            one.wait_stream(two)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))


@pytest.mark.parametrize("layout", ["beside", "behind", "between tokens", "heads first", "one token"])
def test_turned_queries_between_others(gpu, layout):
    """Queries and turned ones in one tensor, whose rows do not meet."""
    import torch
    _say("rotary within one tensor", layout)
    g = torch.Generator(device="cuda").manual_seed(40)
    tokens, heads, kv_heads, dim = 1 if layout == "one token" else 21, 6, 2, 64
    shape = {"beside": (tokens, heads, 2, dim), "behind": (2, tokens, heads, dim), "between tokens": (tokens, 2, heads, dim),
             "heads first": (2, heads, tokens, dim), "one token": (tokens, heads, 2, dim)}[layout]
    both = torch.randn(*shape, device="cuda", generator=g).half()
    axis = shape.index(2)
    q, out = both.select(axis, 0), both.select(axis, 1)
    if layout == "heads first":
        q, out = q.transpose(0, 1), out.transpose(0, 1)
    if layout == "one token":  # whose stride may be any number
        out = out.as_strided(out.shape, (7, out.stride(1), 1))
    k = torch.randn(tokens, kv_heads, dim, device="cuda", generator=g).half()
    caches = [torch.zeros(4, 16, kv_heads, dim, device="cuda").half() for _ in range(2)]
    at = torch.arange(tokens, device="cuda") + 5
    freqs, _ = gpu.rotary_frequencies(dim)
    want, before = torch.empty(tokens, heads, dim, device="cuda").half(), q.clone()
    for to in (want, out):
        gpu.paged_rotary(k, k, at.to(torch.int32), freqs, at, *caches, d_q=q, d_q_out=to)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(q, before)


@pytest.mark.parametrize("apart", ["beside", "behind"])
@pytest.mark.parametrize("kv", [300, 20000])
def test_evicted_rows_between_others(gpu, kv, apart):
    """Rows that are read and written in one tensor, beside one another."""
    import torch
    _say("evict within one tensor", kv, apart)
    rng = np.random.default_rng(41)
    n, page, keep = 3, 16, kv // 3
    room = -(-kv // page) * page
    i32 = dict(dtype=torch.int32, device="cuda")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    shape = (n, 2, room) if apart == "beside" else (2, n, room)
    w, at = torch.zeros(shape, device="cuda"), torch.zeros(shape, **i32)
    split = (lambda t, i: t[:, i]) if apart == "beside" else (lambda t, i: t[i])
    weights, places = rng.random((n, room)).astype(np.float32), np.stack([rng.permutation(room) for _ in range(n)]).astype(np.int32)
    split(w, 0).copy_(cuda(weights))
    split(at, 0).copy_(cuda(places))
    table = torch.arange(n * room // page, **i32).view(n, -1)
    full = lambda x: torch.full((n,), x, **i32)  # noqa: E731
    length, n_moves, counts = full(-9), full(-9), torch.zeros(2, **i32)
    moves, freed = torch.zeros(n, room // 2, 2, **i32), torch.zeros(table.numel(), **i32)
    gpu.paged_evict(split(w, 0), full(kv), full(keep), table, page, split(w, 1), length, moves, n_moves, freed, counts,
                    d_positions=split(at, 0), d_kept=full(kv), d_seen=full(kv), d_positions_out=split(at, 1), sinks=2, recent=9)
    torch.cuda.synchronize()
    assert np.array_equal(split(w, 0).cpu().numpy(), weights) and np.array_equal(split(at, 0).cpu().numpy(), places)
    for r in range(n):
        m, lies, pos, _, _ = test_gpu_evict.evict_oracle(weights[r], places[r], kv, kv, kv, keep, table[r].cpu().numpy(), page,
                                                         table.numel(), 2, 9, np.zeros(n * room, bool))
        assert int(length[r]) == m and np.array_equal(split(w, 1)[r, :m].cpu().numpy(), weights[r][lies])
        assert split(at, 1)[r, :m].tolist() == [pos[i] for i in lies]


@pytest.mark.parametrize("what", ["decode ragged", "chunk"])
def test_weights_between_others(gpu, what):
    """What was there and what is written in one tensor, row beside row."""
    import torch
    _say("weights within one tensor", what)
    p = test_gpu_weights.Problem("bfloat16", *test_gpu_weights.SHAPES[what], seed=42)
    room = p.cols * p.page
    both = torch.full((len(p.kv), 2, room), 7.0, device="cuda")
    both[:, 0] = p.past[:, :room]
    gpu.paged_weights(p.q, p.kc, p.table, p.starts, p.kv_len, p.lse, both[:, 1], d_past=both[:, 0], decay=0.75, scale=p.scale)
    torch.cuda.synchronize()
    assert torch.equal(both[:, 0], p.past[:, :room])
    p.check(gpu, out=both[:, 1].cpu().numpy().astype(np.float64))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("decay", [0.75, 1.0, 0.0])
@pytest.mark.parametrize("max_new", [1, 5000])
@pytest.mark.parametrize("what", ["decode ragged", "chunk", "prompt group 3", "more tokens than positions", "dims 256"])
def test_weights_summed_over_layers(gpu, what, max_new, decay, in_place):
    """continued: what was there counts for every entry, the newest among them, times decay; in place as beside it.  The
    product and the sum are rounded once each at most: 2^-23 of either."""
    _say("weights continued", what, max_new, decay, in_place)
    p = test_gpu_weights.Problem("bfloat16", *test_gpu_weights.SHAPES[what], seed=34)
    alone = p.run(gpu, past=False, max_new=max_new)
    p.check(gpu, past=False, out=alone)
    got = p.run(gpu, decay=decay, max_new=max_new, continued=True, in_place=in_place)
    before = p.past.cpu().numpy().astype(np.float64)
    for r, kv in enumerate(p.kv):
        want = alone[r, :kv] + decay * before[r, :kv]
        assert np.all(np.abs(got[r, :kv] - want) <= 2.0 ** -23 * (want + decay * before[r, :kv])), r
        rest = before[r, kv:] if in_place else np.full(got.shape[1], 7.0)[kv:before.shape[1]]
        assert np.array_equal(got[r, kv:before.shape[1]], rest)


def test_a_step_of_layers_decays_once(gpu):
    """Three layers as a step sums them: what older tokens had counts for decay of it, what each layer adds for all."""
    import torch
    _say("weights of a step's layers")
    layers = [test_gpu_weights.Problem("bfloat16", *test_gpu_weights.SHAPES["chunk"], seed=s) for s in (43, 44, 45)]
    decay, room = 0.5, layers[0].cols * 16
    out = layers[0].past.clone()
    for i, p in enumerate(layers):
        gpu.paged_weights(p.q, p.kc, p.table, p.starts, p.kv_len, p.lse, out, d_past=out, decay=decay if i == 0 else 1.0,
                          continued=i > 0, scale=p.scale)
    torch.cuda.synchronize()
    alone = [p.run(gpu, past=False) for p in layers]
    before, got = layers[0].past.cpu().numpy().astype(np.float64), out.cpu().numpy().astype(np.float64)
    for r, (n, kv) in enumerate(zip(layers[0].new, layers[0].kv)):
        want = sum(a[r, :kv] for a in alone)
        want[:kv - n] += decay * before[r, :kv - n]
        assert np.all(np.abs(got[r, :kv] - want) <= 4 * 2.0 ** -24 * want)  # three sums and a product, rounded once each
        assert np.array_equal(got[r, kv:room], before[r, kv:room])


@pytest.mark.parametrize("kind", ["bitmap", "array"])
def test_pinned_slots_behind_the_universe_that_is_named(gpu, kind):
    """Containers uploaded with a universe that ends before their last key: what they hold counts all the same."""
    import torch
    _say("evict, containers behind the universe", kind)
    page, n_pages, kv, keep = 16, 9000, 480, 200
    rng = np.random.default_rng(46)
    i32 = dict(dtype=torch.int32, device="cuda")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    table = (4096 + rng.permutation(4000)[:30]).astype(np.int32)[None]  # slots of the second container
    pinned = np.zeros(n_pages * page, bool)
    slots = (table[0, ::3, None].astype(np.int64) * page + np.arange(0, page, 2)).reshape(-1)
    pinned[slots] = True
    low = np.sort(slots - 65536).astype(np.uint16)
    if kind == "bitmap":
        words = np.zeros(65536, np.uint8)
        words[low] = 1
        first, second = np.zeros(1024, np.uint64), np.packbits(words, bitorder="little").view(np.uint64)
        first[0] = 1
        containers = [(0, gpu.TC_BITSET, 1, first), (1, gpu.TC_BITSET, len(low), second)]
    else:
        containers = [(0, gpu.TC_ARRAY, 1, np.zeros(1, np.uint16)), (1, gpu.TC_ARRAY, len(low), low)]
    g = gpu.upload_containers(containers, universe=1000, threshold=gpu.PROMOTE_KEEP_DEFAULT)
    assert g.n_bitmap_containers == (2 if kind == "bitmap" else 0)
    pinned[0] = True
    w = rng.random((1, 480)).astype(np.float32)
    one = lambda x: torch.tensor([x], **i32)  # noqa: E731
    out, length, n_moves = torch.zeros(1, 480, device="cuda"), one(-9), one(-9)
    moves, freed, counts = torch.full((1, 240, 2), -9, **i32), torch.full((30,), -9, **i32), torch.zeros(2, **i32)
    gpu.paged_evict(cuda(w), one(kv), one(keep), cuda(table), page, out, length, moves, n_moves, freed, counts, sinks=2,
                    recent=4, pinned=g, n_pages=n_pages)
    torch.cuda.synchronize()
    gpu.free(g)
    m, lies, _, want, _ = test_gpu_evict.evict_oracle(w[0], w[0], 0, kv, kv, keep, table[0], page, n_pages, 2, 4, pinned)
    assert int(length[0]) == m and int(n_moves[0]) == len(want) > 0
    assert moves[0, :len(want)].tolist() == [list(x) for x in want]
    assert np.array_equal(out[0, :m].cpu().numpy(), w[0][lies])
