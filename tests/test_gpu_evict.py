"""paged_evict and paged_move against plain loops over the same entries, bit by bit."""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


def evict_oracle(weights, positions, kept, seen, kv, keep, table, page, n_pages, sinks, recent, pinned):
    """Of one request: (m, the entries in the order in which they then lie, moves as (from, to) slots, columns freed)."""
    room = table.shape[0] * page
    n = min(max(0, kv), room)
    kept = min(max(0, kept), n)
    pos = [int(positions[i]) if i < kept else seen - n + i for i in range(n)]

    def slot(i):
        p = int(table[i // page])
        return p * page + i % page if 0 <= p < n_pages else -1

    safe = [pos[i] < sinks or pos[i] >= seen - recent or (slot(i) >= 0 and bool(pinned[slot(i)])) for i in range(n)]
    m = max(min(n, max(0, keep)), sum(safe))
    weight = [-np.inf if np.isnan(w) else float(w) for w in weights[:n]]
    order = sorted(range(n), key=lambda i: (not safe[i], bool(np.isnan(weights[i])) if not safe[i] else False,
                                            -weight[i] if not safe[i] else 0.0, i))
    stay = set(order[:m])
    holes = [i for i in range(m) if i not in stay]
    movers = [i for i in range(m, n) if i in stay]
    assert len(holes) == len(movers)
    lies = list(range(m))
    for h, s in zip(holes, movers):
        lies[h] = s
    moves = [(slot(s), slot(h)) for h, s in zip(holes, movers)]
    return m, lies, pos, moves, list(range(-(-m // page), -(-n // page)))


class Problem:
    def __init__(self, kv, keep, page=16, seed=0, sinks=2, recent=8, pinned=None, kept=None, weights="spread", wide=0,
                 seen_more=3):
        import torch
        rng = np.random.default_rng(seed)
        self.kv, self.page, self.sinks, self.recent = np.asarray(kv, np.int32), page, sinks, recent
        n = len(kv)
        self.keep = np.asarray(keep, np.int32)
        held = [-(-max(0, int(x)) // page) for x in kv]
        self.cols = max(1, max(held)) + wide
        self.pages = sum(held) + 5
        order = rng.permutation(self.pages)
        self.table = np.full((n, self.cols), -1, np.int32)
        at = 0
        for r, h in enumerate(held):
            self.table[r, :h] = order[at:at + h]
            at += h
        room = self.cols * page
        w = rng.standard_normal((n, room)).astype(np.float32)
        if weights == "spread":
            w = np.exp(3 * w).astype(np.float32)
        elif weights == "alike":
            w = np.round(w).astype(np.float32)
        elif weights == "same":
            w = np.full((n, room), 0.25, np.float32)
        elif weights == "odd":
            w[rng.random((n, room)) < 0.2] = np.nan
            w[rng.random((n, room)) < 0.2] = np.inf
            w[rng.random((n, room)) < 0.2] = -np.inf
            w[rng.random((n, room)) < 0.2] = 0.0
            w[rng.random((n, room)) < 0.2] = -0.0
        self.weights = w
        self.kept = np.asarray([rng.integers(0, max(0, int(x)) + 1) for x in kv] if kept is None else kept, np.int32)
        self.seen = (np.maximum(self.kv, 0) + seen_more).astype(np.int32)
        self.positions = np.stack([rng.permutation(room) for _ in range(n)]).astype(np.int32)
        self.pinned = np.zeros(self.pages * page, bool) if pinned is None else rng.random(self.pages * page) < pinned
        self.torch = torch

    def check(self, gpu, kind="bitmap", positions=True, in_place=False, pad=0, stream=None, freed_cap=None, heads=2, dim=8,
              dtype="float16"):
        torch, n, room = self.torch, len(self.kv), self.cols * self.page
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        i32 = dict(dtype=torch.int32, device="cuda")

        def padded(a, fill):
            t = torch.full((n, room + pad), fill, dtype=torch.float32 if a.dtype == np.float32 else torch.int32, device="cuda")
            t[:, :room] = cuda(a)
            return t

        weights, places = padded(self.weights, 7.0), padded(self.positions, -7)
        w_out = weights if in_place else torch.full((n, room + pad), 9.0, device="cuda")
        p_out = places if in_place else torch.full((n, room + pad), -9, **i32)
        length, n_moves, counts = torch.full((n,), -9, **i32), torch.full((n,), -9, **i32), torch.full((2,), -9, **i32)
        moves = torch.full((n, room // 2 + 2, 2), -9, **i32)
        cap = self.pages if freed_cap is None else freed_cap
        freed = torch.full((cap + 3,), -9, **i32)
        g = None
        if self.pinned.any() or kind != "bitmap":
            g = gpu.upload_from_ids(np.nonzero(self.pinned)[0].astype(np.uint32), self.pinned.size,
                                    gpu.PROMOTE_ALL if kind == "bitmap" else gpu.PROMOTE_KEEP_DEFAULT)
        gpu.paged_evict(weights, cuda(self.kv), cuda(self.keep), cuda(self.table), self.page, w_out, length, moves, n_moves,
                        freed[:cap], counts, d_positions=places if positions else None,
                        d_kept=cuda(self.kept) if positions else None, d_seen=cuda(self.seen) if positions else None,
                        d_positions_out=p_out, sinks=self.sinks, recent=self.recent, pinned=g, n_pages=self.pages,
                        stream=stream)
        dt = getattr(torch, dtype)
        gen = torch.Generator(device="cuda").manual_seed(3)
        kc = torch.randn(self.pages, self.page, heads, dim, device="cuda", generator=gen).to(dt)
        vc = torch.randn(self.pages, self.page, heads, dim, device="cuda", generator=gen).to(dt)
        k0, v0 = kc.clone(), vc.clone()
        gpu.paged_move(moves, n_moves, kc, vc, stream=stream)
        torch.cuda.synchronize()
        if g is not None:
            gpu.free(g)
        host = lambda t: t.cpu().numpy()  # noqa: E731
        all_freed, all_moves = [], 0
        w_got, p_got, moves, n_moves = host(w_out), host(p_out), host(moves), host(n_moves)
        for r in range(n):
            kv = int(self.kv[r])
            m, lies, pos, want, cols = evict_oracle(
                self.weights[r], self.positions[r], int(self.kept[r]) if positions else 0,
                int(self.seen[r]) if positions else max(0, min(kv, room)), kv, int(self.keep[r]), self.table[r], self.page,
                self.pages, self.sinks, self.recent, self.pinned)
            assert int(length[r]) == m and int(n_moves[r]) == len(want), (r, int(length[r]), m, int(n_moves[r]), len(want))
            assert moves[r, :len(want)].tolist() == [list(x) for x in want], r
            assert np.all(moves[r, len(want):] == -9)
            assert np.array_equal(w_got[r, :m], self.weights[r][lies], equal_nan=True)
            assert p_got[r, :m].tolist() == [pos[i] for i in lies]
            if in_place:
                assert np.array_equal(w_got[r, m:room], self.weights[r, m:], equal_nan=True)
                assert np.array_equal(p_got[r, m:room], self.positions[r, m:])
            else:
                assert np.all(w_got[r, m:] == 9.0) and np.all(p_got[r, m:] == -9)
            all_freed += [int(self.table[r, c]) for c in cols]
            all_moves += len(want)
            for a, b in want:
                if a >= 0 and b >= 0:
                    k0.view(-1, heads, dim)[b], v0.view(-1, heads, dim)[b] = (t.view(-1, heads, dim)[a] for t in (kc, vc))
        assert host(counts).tolist() == [len(all_freed), all_moves]
        assert host(freed)[:min(cap, len(all_freed))].tolist() == all_freed[:cap]
        assert np.all(host(freed)[min(cap, len(all_freed)):] == -9)
        assert torch.equal(kc, k0) and torch.equal(vc, v0)


LENGTHS = {
    "one": ([40], [20]), "nothing to do": ([40, 7], [40, 100]), "ragged": ([1, 100, 257, 64, 0], [1, 30, 200, 0, 5]),
    "one goes": ([300, 17], [299, 16]), "all go but the safe": ([200, 90], [0, -5]), "negative": ([-4, 30], [3, 10]),
    "many": (list(range(1, 70)), list(range(69, 0, -1))), "a page": ([16, 32], [15, 17]),
}


@pytest.mark.parametrize("weights", ["spread", "alike", "same", "odd"])
@pytest.mark.parametrize("what", LENGTHS)
def test_evict(gpu, what, weights):
    _say("evict", what, weights)
    Problem(*LENGTHS[what], seed=len(what), weights=weights).check(gpu)


@pytest.mark.parametrize("kind", ["bitmap", "arrays"])
@pytest.mark.parametrize("pinned", [0.0, 0.1, 0.9, 1.0])
@pytest.mark.parametrize("what", ["ragged", "many", "all go but the safe"])
def test_evict_with_pinned_slots(gpu, what, pinned, kind):
    _say("evict pinned", what, pinned, kind)
    Problem(*LENGTHS[what], seed=2, pinned=pinned).check(gpu, kind)


@pytest.mark.parametrize("what", [dict(sinks=0, recent=0), dict(sinks=1 << 30, recent=0), dict(sinks=0, recent=1 << 30),
                                  dict(page=1), dict(page=256), dict(wide=3), dict(seen_more=0), dict(seen_more=100000),
                                  dict(kept=[0] * 5), dict(kept=[10 ** 6] * 5), dict(kept=[-3] * 5)])
def test_evict_edges(gpu, what):
    _say("evict", what)
    Problem(*LENGTHS["ragged"], seed=3, **what).check(gpu)
    Problem(*LENGTHS["ragged"], seed=3, weights="alike", **what).check(gpu, in_place=True, pad=3)


def test_evict_by_places(gpu):
    _say("evict without positions")
    Problem(*LENGTHS["ragged"], seed=4).check(gpu, positions=False)


def test_evict_short_list_of_freed_pages(gpu):
    _say("evict with room for few freed pages")
    for cap in (0, 1, 5):
        Problem(*LENGTHS["ragged"], seed=5).check(gpu, freed_cap=cap)


@pytest.mark.parametrize("dtype,heads,dim", [("float32", 1, 64), ("bfloat16", 3, 80), ("float16", 1, 3), ("float32", 2, 1),
                                             ("bfloat16", 8, 128)])
def test_move_types(gpu, dtype, heads, dim):
    _say("move", dtype, heads, dim)
    Problem(*LENGTHS["ragged"], seed=6).check(gpu, dtype=dtype, heads=heads, dim=dim)


@pytest.mark.parametrize("kv,keep", [([4095, 4096, 4097], [1000, 4000, 4096]), ([20011], [5000]), ([9000] * 3, [8999, 4500, 1])])
def test_evict_long(gpu, kv, keep):
    _say("evict long", kv, keep)
    Problem(kv, keep, seed=7, pinned=0.05, recent=100).check(gpu)
    Problem(kv, keep, seed=8, weights="alike", recent=100).check(gpu, in_place=True)


@pytest.mark.parametrize("weights", ["spread", "alike", "same", "odd"])
@pytest.mark.parametrize("what", LENGTHS)
def test_evict_short_requests_in_long_rows(gpu, what, weights):
    """Rows with room for more than one workgroup looks at."""
    _say("evict in long rows", what, weights)
    Problem(*LENGTHS[what], seed=len(what), weights=weights, wide=1100, pinned=0.1).check(gpu)


@pytest.mark.parametrize("weights", ["spread", "alike", "same", "odd"])
@pytest.mark.parametrize("page", [1, 2, 64])
def test_evict_long_rows_of_every_kind(gpu, weights, page):
    _say("evict long rows", weights, page)
    p = Problem([17000, 16385, 9000, 4096, 4097], [9000, 16384, 0, 4000, 10 ** 6], seed=13, weights=weights, page=page,
                pinned=0.02, recent=77)
    p.check(gpu)
    p.check(gpu, in_place=True, pad=5)


@pytest.mark.parametrize("weights", ["spread", "alike"])
@pytest.mark.parametrize("room", [1008, 1024, 1040, 2048, 2064, 4096, 4112, 8192])
def test_evict_rooms(gpu, room, weights):
    """As many positions as the kernels of each size hold, and one page more."""
    _say("evict room", room, weights)
    Problem([room], [room // 3], seed=room, weights=weights, pinned=0.05).check(gpu)
    Problem([room - 5, 3, room, 40], [room // 2, 1, room - 1, 100], seed=room + 1, weights=weights).check(gpu, in_place=True)


def test_evict_very_long(gpu):
    _say("evict very long")
    Problem([70001, 131072], [30000, 120000], seed=9, page=64, recent=500, pinned=0.01).check(gpu)


@pytest.mark.parametrize("kinds,keep", [(100, 1500000), (100, 40), (2, 2150000), (1 << 30, 3000000)])
def test_evict_millions(gpu, kinds, keep):
    """A row of more segments than a workgroup's waves have lanes, with ties across them."""
    import torch
    _say("evict millions", kinds, keep)
    rng = np.random.default_rng(kinds % 97)
    n, page, sinks, recent = 4300003, 64, 3, 1000
    cols = -(-n // page)
    table = rng.permutation(cols).astype(np.int32)
    w = rng.integers(0, kinds, cols * page).astype(np.float32)
    i32 = dict(dtype=torch.int32, device="cuda")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    one = lambda x: torch.tensor([x], **i32)  # noqa: E731
    w_out, length, n_moves, counts = torch.zeros(1, cols * page, device="cuda"), one(-9), one(-9), torch.zeros(2, **i32)
    moves, freed = torch.full((1, cols * page // 2, 2), -9, **i32), torch.full((cols,), -9, **i32)
    gpu.paged_evict(cuda(w)[None], one(n), one(keep), cuda(table)[None], page, w_out, length, moves, n_moves, freed, counts,
                    sinks=sinks, recent=recent)
    place = np.arange(n)
    safe = (place < sinks) | (place >= n - recent)
    keep = max(keep, int(safe.sum()))
    stay = np.zeros(n, bool)
    stay[np.lexsort((place, -w[:n], ~safe))[:keep]] = True
    holes, movers = np.nonzero(~stay[:keep])[0], keep + np.nonzero(stay[keep:])[0]
    slot = lambda i: table[i // page] * page + i % page  # noqa: E731
    lies = np.arange(keep)
    lies[holes] = movers
    assert int(length[0]) == keep and int(n_moves[0]) == len(holes)
    assert np.array_equal(moves[0, :len(holes)].cpu().numpy(), np.stack([slot(movers), slot(holes)], 1))
    assert np.array_equal(w_out[0, :keep].cpu().numpy(), w[lies])
    first = -(-keep // page)
    assert counts.tolist() == [cols - first, len(holes)]
    assert np.array_equal(freed[:cols - first].cpu().numpy(), table[first:])


def test_a_page_outside_the_cache(gpu):
    """Its entries can not be pinned; a move from or to it is listed as -1 and left out."""
    _say("evict with pages outside the cache")
    p = Problem([100, 100], [30, 60], seed=10, pinned=0.3)
    p.table[0, 1], p.table[1, 5] = -1, p.pages
    p.check(gpu)


def test_another_stream(gpu):
    import torch
    _say("evict on another stream")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        Problem(*LENGTHS["many"], seed=11, pinned=0.1).check(gpu, stream=s)


def test_no_requests(gpu):
    import torch
    _say("evict without requests")
    i32 = dict(dtype=torch.int32, device="cuda")
    none, counts = torch.zeros(0, **i32), torch.full((2,), 9, **i32)
    gpu.paged_evict(torch.zeros(0, 16, device="cuda"), none, none, torch.zeros(0, 1, **i32), 16, torch.zeros(0, 16, device="cuda"),
                    none, torch.zeros(0, 8, 2, **i32), none, none, counts)
    c = torch.ones(2, 16, 1, 8, device="cuda")
    gpu.paged_move(torch.zeros(0, 8, 2, **i32), none, c, c.clone())
    torch.cuda.synchronize()
    assert counts.tolist() == [0, 0]


def test_moves_of_noise_stay_inside(gpu):
    import torch
    _say("moves of noise")
    g = torch.Generator(device="cuda").manual_seed(1)
    held = torch.zeros(12, 16, 2, 8, device="cuda", dtype=torch.float16)
    kc, vc = held[2:6], held[8:11 + 1][:4]
    kc.fill_(1.0)
    vc.fill_(1.0)
    for i in range(10):
        moves = torch.randint(-2 ** 31, 2 ** 31 - 1, (3, 9, 2), generator=g, device="cuda").to(torch.int32)
        n = torch.randint(-2 ** 31, 2 ** 31 - 1, (3,), generator=g, device="cuda").to(torch.int32)
        gpu.paged_move(moves, n, kc, vc)
    torch.cuda.synchronize()
    assert torch.all(held[:2] == 0) and torch.all(held[6:8] == 0) and torch.all(kc == 1) and torch.all(vc == 1)


def test_evictions_in_a_row(gpu):
    """A request that grows and is cut again and again: the sinks, the last tokens and the heaviest are there in the end,
    under their own positions."""
    import torch
    _say("evict again and again")
    rng = np.random.default_rng(12)
    page, cols, keep, sinks, recent = 8, 20, 60, 3, 10
    room = cols * page
    i32 = dict(dtype=torch.int32, device="cuda")
    weights, positions = torch.zeros(1, room, device="cuda"), torch.zeros(1, room, **i32)
    weight_of, length, kept, seen = {}, 0, 0, 0
    table = torch.arange(cols, **i32)[None]
    moves, n_moves, counts = torch.zeros(1, room // 2, 2, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32)
    freed, out = torch.zeros(cols, **i32), torch.zeros(1, **i32)
    cache = torch.zeros(cols, page, 1, 1, device="cuda")
    for _ in range(12):
        new = int(rng.integers(1, 50))
        for i in range(new):
            w = float(np.float32(rng.random()))
            weight_of[seen + i] = w
            weights[0, length + i] = w
            cache.view(-1)[length + i] = seen + i
        length, seen = length + new, seen + new
        now = lambda x: torch.tensor([x], **i32)  # noqa: E731
        gpu.paged_evict(weights, now(length), now(keep), table, page, weights, out, moves, n_moves, freed, counts,
                        d_positions=positions, d_kept=now(kept), d_seen=now(seen), d_positions_out=positions, sinks=sinks,
                        recent=recent, n_pages=cols)
        gpu.paged_move(moves, n_moves, cache, cache.clone())
        torch.cuda.synchronize()
        length = kept = int(out[0])
        there = positions[0, :length].tolist()
        assert cache.view(-1)[:length].tolist() == [float(x) for x in there]
        assert len(set(there)) == length == min(seen, keep)
        assert set(range(sinks)) <= set(there) and set(range(max(0, seen - recent), seen)) <= set(there)
        assert weights[0, :length].tolist() == [weight_of[p] for p in there]
        weight_of = {p: weight_of[p] for p in there}
