"""The paged cache's bookkeeping: paged_plan, paged_append and paged_select
against plain loops over the same lengths, bit-exact."""
import numpy as np
import pytest

import orc  # noqa: F401  (the oracle's folder is on the path of every GPU test)

pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


def _cuda(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _bitmap(gpu, mask, kind="bitmap"):
    """The set of `mask` in a layout: bitmaps, arrays, stored as its complement, or with runs."""
    ids = np.nonzero(mask)[0].astype(np.uint32)
    n = len(mask)
    if kind == "bitset":
        words = np.zeros((n + 31) // 32, np.uint32)
        np.bitwise_or.at(words, ids // 32, np.uint32(1) << (ids % 32).astype(np.uint32))
        return gpu.upload_from_bitset(words, n)
    g = gpu.upload_from_ids(ids, n, gpu.PROMOTE_ALL if kind == "bitmap" else gpu.PROMOTE_KEEP_DEFAULT)
    if kind == "stored":  # arrays, bitmaps and runs as the portable format chooses them
        s = gpu.portable_serialize(g)
        gpu.free(g)
        return gpu.portable_deserialize(s, n, gpu.PROMOTE_KEEP_DEFAULT)
    return g


# ---- plan ------------------------------------------------------------------------
def plan_oracle(free, page, cached, new, table, slots_cap, taken_cap):
    ids = np.nonzero(free)[0].tolist()
    table, n = table.copy(), len(cached)
    slots, starts, kv_len, taken = [], [0], [], []
    upto = missing = 0
    for r in range(n):
        c, m = int(cached[r]), int(new[r])
        tokens = max(m, 0)
        held, most = -(-max(c, 0) // page), -(-(max(c, 0) + tokens) // page)
        fits = c >= 0 and m >= 0 and most <= table.shape[1]
        need = most - held if fits else 0
        granted = fits and (need == 0 or upto + need <= len(ids))
        upto += need
        if granted:
            for i in range(need):
                table[r, held + i] = ids[upto - need + i]
                taken.append(ids[upto - need + i])
        elif most > held:
            missing += most - held
        kv_len.append(c + m if granted else 0)
        for i in range(tokens):
            slots.append(int(table[r, (c + i) // page]) * page + (c + i) % page if granted and c + m > 0 else -1)
        starts.append(starts[-1] + tokens)
    return table, slots[:slots_cap], starts, kv_len, taken[:taken_cap], [starts[-1], len(taken), missing]


def check_plan(gpu, free, page, cached, new, cols, kind="bitmap", slots_cap=None, taken_cap=None, pad=0):
    import torch
    n, pages = len(cached), len(free)
    rng = np.random.default_rng(5)
    busy = np.nonzero(~free)[0]
    table = np.full((n, cols), -1, np.int32)
    for r in range(n):
        held = min(cols, max(0, -(-int(cached[r]) // page)))
        if held and busy.size:
            table[r, :held] = rng.choice(busy, held)
    total = int(np.maximum(new, 0).sum())
    slots_cap = total if slots_cap is None else slots_cap
    taken_cap = pages if taken_cap is None else taken_cap
    want = plan_oracle(free, page, cached, new, table, slots_cap, taken_cap)
    g = _bitmap(gpu, free, kind)
    wide = torch.full((n, cols + pad), -7, dtype=torch.int32, device="cuda")
    d_table = wide[:, :cols]
    d_table.copy_(_cuda(table))
    d_slots = torch.full((slots_cap + 3,), -9, dtype=torch.int64, device="cuda")
    d_taken = torch.full((taken_cap + 3,), -9, dtype=torch.int32, device="cuda")
    d_starts = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda")
    d_kv = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    d_counts = torch.full((3,), -9, dtype=torch.int32, device="cuda")
    gpu.paged_plan(g, pages, page, _cuda(np.asarray(cached, np.int32)), _cuda(np.asarray(new, np.int32)), d_table,
                   d_slots[:slots_cap], d_starts, d_kv, d_taken[:taken_cap], d_counts)
    torch.cuda.synchronize()
    gpu.free(g)
    assert np.array_equal(d_table.cpu().numpy(), want[0])
    assert np.array_equal(d_starts.cpu().numpy(), want[2])
    assert np.array_equal(d_kv.cpu().numpy(), want[3])
    assert np.array_equal(d_counts.cpu().numpy(), want[5])
    s, t = d_slots.cpu().numpy(), d_taken.cpu().numpy()
    assert np.array_equal(s[:len(want[1])], want[1]) and np.all(s[len(want[1]):] == -9)
    assert np.array_equal(t[:len(want[4])], want[4]) and np.all(t[len(want[4]):] == -9)
    assert np.all(wide.cpu().numpy()[:, cols:] == -7)


@pytest.mark.parametrize("kind", ["bitmap", "arrays", "bitset", "stored"])
@pytest.mark.parametrize("requests,pages,page", [(1, 40, 16), (64, 5000, 16), (1100, 9001, 8), (300, 70001, 1),
                                                 (7, 200003, 128)])
def test_plan(gpu, kind, requests, pages, page):
    _say("plan", kind, requests, pages, page)
    rng = np.random.default_rng(pages)
    share = pages * page // (3 * requests)
    cached = rng.integers(0, min(share, 900) + 1, requests)
    new = rng.integers(0, min(share, 900) + 1, requests)
    free = rng.random(pages) < 0.7
    cols = int((cached + new + page - 1).max() // page) + 1
    check_plan(gpu, free, page, cached, new, cols, kind, pad=5)


def test_plan_edges(gpu):
    rng = np.random.default_rng(1)
    free = rng.random(3000) < 0.5
    for what, cached, new, cols in (
            ("no new tokens", [5, 0, 16], [0, 0, 0], 4),
            ("at a page's end", [16, 15, 17, 0], [1, 1, 15, 16], 4),
            ("negative lengths are refused", [-1, 5, 7], [4, -3, 2], 4),
            ("rows too short are refused", [10, 10, 60], [200, 6, 4], 4),
            ("one request", [0], [1], 1)):
        _say("plan", what)
        check_plan(gpu, free, 16, np.array(cached), np.array(new), cols)


def test_plan_runs_out_of_pages(gpu):
    """In order: later requests that need no page still go through, and nothing is taken for the refused."""
    _say("plan without enough pages")
    free = np.zeros(500, bool)
    free[[3, 77, 78, 410, 499]] = True
    check_plan(gpu, free, 16, np.array([0, 4, 16, 0, 3, 30]), np.array([33, 2, 17, 40, 5, 2]), 8)
    check_plan(gpu, np.zeros(500, bool), 16, np.array([0, 4]), np.array([1, 2]), 8)
    check_plan(gpu, np.ones(1, bool), 16, np.array([0, 0]), np.array([16, 1]), 8)


def test_plan_buffers_bound_what_is_written(gpu):
    _say("plan with short slot and page lists")
    rng = np.random.default_rng(2)
    check_plan(gpu, rng.random(4000) < 0.5, 16, rng.integers(0, 90, 40), rng.integers(1, 300, 40), 30, slots_cap=1001,
               taken_cap=17)


def test_plan_then_take_and_give_back(gpu):
    """The ids taken leave the free set and come back to it through the set operations."""
    import torch
    _say("plan, take, give back")
    free = np.random.default_rng(3).random(5000) < 0.5
    g = _bitmap(gpu, free)
    i32 = dict(dtype=torch.int32, device="cuda")
    table, starts, kv, counts = (torch.full((4, 40), -1, **i32), torch.zeros(5, **i32), torch.zeros(4, **i32),
                                 torch.zeros(3, **i32))
    slots, taken = torch.zeros(400, dtype=torch.int64, device="cuda"), torch.full((100,), -1, **i32)
    new = torch.tensor([100, 1, 170, 129], **i32)
    gpu.paged_plan(g, 5000, 16, torch.zeros(4, **i32), new, table, slots, starts, kv, taken, counts)
    torch.cuda.synchronize()
    n = int(counts[1])
    assert n == 7 + 1 + 11 + 9
    t = gpu.upload_from_device_ids(taken[:n].contiguous(), 5000)
    left = gpu.set_operation(g, t, gpu.ANDNOT)
    assert gpu.cardinality(left) == int(free.sum()) - n
    back = gpu.set_operation(left, t, gpu.OR)
    words = torch.zeros((5000 + 31) // 32, **i32)
    gpu.decompress_to_bitset(back, words)
    torch.cuda.synchronize()
    bits = np.unpackbits(words.cpu().numpy().view(np.uint8), bitorder="little")[:5000]
    assert np.array_equal(bits.astype(bool), free)
    for x in (g, t, left, back):
        gpu.free(x)


# ---- append ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 8, 1), (5, 3, 64, 16), (700, 8, 128, 16), (333, 2, 80, 64),
                                                   (50, 3, 20, 4), (9, 1, 5, 8)])
def test_append(gpu, dtype, tokens, heads, dim, page):
    import torch
    _say("append", dtype, tokens, heads, dim, page)
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    k, v = (torch.randn(tokens, heads, dim, device="cuda", generator=g).to(dt) for _ in range(2))
    kc, vc = (torch.randn(pages, page, heads, dim, device="cuda", generator=g).to(dt) for _ in range(2))
    if tokens > 4:  # left out
        slots[1], slots[3] = -1, pages * page
    want_k, want_v = kc.clone(), vc.clone()
    ok = (slots >= 0) & (slots < pages * page)
    want_k.view(-1, heads, dim)[slots[ok]] = k[ok]
    want_v.view(-1, heads, dim)[slots[ok]] = v[ok]
    gpu.paged_append(k, v, slots, kc, vc)
    torch.cuda.synchronize()
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.parametrize("layout", ["heads first", "padded rows", "offset by one"])
def test_append_strides(gpu, layout):
    """Caches and inputs that are views: pages of [heads, slots], rows with room between them, odd addresses."""
    import torch
    _say("append strides", layout)
    tokens, heads, dim, page, pages = 77, 4, 64, 16, 9
    g = torch.Generator(device="cuda").manual_seed(4)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    if layout == "heads first":
        kc, vc = (new(pages, heads, page, dim).transpose(1, 2) for _ in range(2))
        qkv = new(tokens, 3 * heads, dim)
        k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    elif layout == "padded rows":
        kc, vc = (new(pages, page, heads, dim + 24)[..., 8:8 + dim] for _ in range(2))
        k, v = (new(heads, tokens, dim).transpose(0, 1) for _ in range(2))
    else:
        kc, vc = (new(pages * page * heads * dim + 1)[1:].view(pages, page, heads, dim) for _ in range(2))
        k, v = (new(tokens * heads * dim + 1)[1:].view(tokens, heads, dim) for _ in range(2))
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    want = [c.clone() for c in (kc, vc)]
    for w, x in zip(want, (k, v)):
        w[slots // page, slots % page] = x
    gpu.paged_append(k, v, slots, kc, vc)
    torch.cuda.synchronize()
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


# ---- select ----------------------------------------------------------------------
def select_oracle(visible, table, starts, kv_len, page, n_pages):
    sel, limits = [], np.full(int(starts[-1]), -5, np.int32)
    for r in range(len(kv_len)):
        length = min(max(int(kv_len[r]), 0), table.shape[1] * page)
        pages = table[r, np.arange(length) // page].astype(np.int64)
        slots = pages * page + np.arange(length) % page
        ok = (pages >= 0) & (pages < n_pages)
        ok[ok] = visible[slots[ok]]
        sel.append(slots[ok])
        upto = np.concatenate([[0], np.cumsum(ok)])
        n = int(starts[r + 1] - starts[r])
        for i in range(n):
            limits[starts[r] + i] = upto[max(0, length - n + i + 1)]
    return sel, limits


@pytest.mark.parametrize("density", [0.0, 0.03, 0.5, 1.0])
@pytest.mark.parametrize("page,pages,kv,new", [(16, 900, [1, 700, 33, 0, 64], [1, 5, 33, 0, 2]),
                                               (64, 700, [20000, 8192, 8193], [1, 300, 1]),
                                               (1, 500, [100, 31], [100, 40]), (8, 90, [5], [9]), (32, 1500, [40000], [9000])])
def test_select(gpu, density, page, pages, kv, new):
    import torch
    _say("select", density, page, pages, kv)
    rng = np.random.default_rng(pages)
    cols = max(1, max(-(-x // page) for x in kv))
    table = rng.integers(0, pages, (len(kv), cols)).astype(np.int32)
    if page == 16:
        table[1, 3], table[1, 5] = -1, pages  # pages outside the cache are not visible
    visible = rng.random(pages * page) < density
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    for kind in ("bitmap", "stored"):
        g = _bitmap(gpu, visible, kind)
        i32 = dict(dtype=torch.int32, device="cuda")
        sel, length = torch.full((len(kv), cols * page + 2), -5, **i32), torch.full((len(kv),), -5, **i32)
        limits = torch.full((int(starts[-1]),), -5, **i32)
        gpu.paged_select(g, _cuda(table), _cuda(starts), _cuda(np.array(kv, np.int32)), page, sel, length, limits, pages)
        torch.cuda.synchronize()
        gpu.free(g)
        want, want_limits = select_oracle(visible, table, starts, np.array(kv), page, pages)
        assert np.array_equal(length.cpu().numpy(), [len(x) for x in want])
        for r, x in enumerate(want):
            row = sel[r].cpu().numpy()
            assert np.array_equal(row[:len(x)], x) and np.all(row[len(x):] == -5)
        assert np.array_equal(limits.cpu().numpy(), want_limits)


@pytest.mark.parametrize("kind", ["bitmap", "stored"])
@pytest.mark.parametrize("page,pages,kv,new", [(64, 1100, [32768, 2049, 32767, 0], [2050, 1, 64, 0]),
                                               (64, 600, [32769, 32705], [1, 4097]),
                                               (16, 2100, [16384, 4097, 2048, 4096], [3, 4097, 2048, 1]),
                                               (8, 1200, [8192, 6145, 1], [40, 2047, 1]),
                                               (2, 3000, [2050, 2048, 2047], [2050, 2, 1]),
                                               (128, 300, [30001, 16385], [33, 2])])
def test_select_counts_chunks(gpu, page, pages, kv, new, kind):
    """Requests of several chunks, up to and above the look-ups that a workgroup makes by itself; some pages outside."""
    import torch
    _say("select chunks", page, pages, kv, kind)
    rng = np.random.default_rng(page)
    cols = max(-(-x // page) for x in kv)
    table = rng.integers(-3, pages + 3, (len(kv), cols)).astype(np.int32)
    visible = rng.random(pages * page) < 0.4
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    g = _bitmap(gpu, visible, kind)
    i32 = dict(dtype=torch.int32, device="cuda")
    sel, length = torch.full((len(kv), cols * page + 2), -5, **i32), torch.full((len(kv),), -5, **i32)
    limits = torch.full((int(starts[-1]),), -5, **i32)
    gpu.paged_select(g, _cuda(table), _cuda(starts), _cuda(np.array(kv, np.int32)), page, sel, length, limits, pages)
    torch.cuda.synchronize()
    gpu.free(g)
    want, want_limits = select_oracle(visible, table, starts, np.array(kv), page, pages)
    assert np.array_equal(length.cpu().numpy(), [len(x) for x in want])
    for r, x in enumerate(want):
        row = sel[r].cpu().numpy()
        assert np.array_equal(row[:len(x)], x) and np.all(row[len(x):] == -5)
    assert np.array_equal(limits.cpu().numpy(), want_limits)


@pytest.mark.parametrize("page,cols,kv,new", [(16, 3, [55, 48, 200, 30, 49, -4, 0], [10, 4, 70, 3, 1, 2, 2]),
                                              (64, 70, [4490, 9000], [30, 4600]), (2, 1100, [2205, 2201], [2205, 1])])
@pytest.mark.parametrize("density", [0.4, 1.0])
def test_select_of_requests_longer_than_the_table(gpu, page, cols, kv, new, density):
    """A token's place is by its request's length, also where the table does not hold all of it, as attention has it."""
    import torch
    _say("select past the table", page, cols, kv)
    rng = np.random.default_rng(cols)
    n, pages, room = len(kv), 2 * cols, cols * page
    table = np.stack([rng.permutation(pages)[:cols] for _ in range(n)]).astype(np.int32)
    visible = rng.random(pages * page) < density
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    want, want_len = [], []
    for r in range(n):
        pos = np.arange(min(room, max(0, kv[r])))
        upto = np.concatenate([[0], np.cumsum(visible[table[r, pos // page].astype(np.int64) * page + pos % page])])
        want_len.append(upto[-1])
        want += [upto[min(len(pos), max(0, kv[r] - new[r] + i + 1))] for i in range(new[r])]
    g = _bitmap(gpu, visible)
    i32 = dict(dtype=torch.int32, device="cuda")
    sel, length, limits = torch.zeros(n, room, **i32), torch.full((n,), -5, **i32), torch.full((len(want) + 2,), -5, **i32)
    lens = _cuda(np.array(kv, np.int32))
    gpu.paged_select(g, _cuda(table), _cuda(starts), lens, page, sel, length, limits[:-2], pages)
    torch.cuda.synchronize()
    gpu.free(g)
    assert np.array_equal(length.cpu().numpy(), want_len)
    assert np.array_equal(limits.cpu().numpy(), want + [-5, -5])
    if density == 1.0:  # all is visible: the answers of attention without a selection, to the order of its sums
        gen = torch.Generator(device="cuda").manual_seed(1)
        q, kc, vc = (torch.randn(*s, device="cuda", generator=gen).half() for s in ((len(want), 2, 64), (pages, page, 1, 64),
                                                                                  (pages, page, 1, 64)))
        out = [torch.full_like(q, 7.0) for _ in range(2)]
        for o, chosen in zip(out, (None, (sel, length, limits[:-2].contiguous()))):
            gpu.paged_attention(q, kc, vc, _cuda(table), _cuda(starts), lens, o, selection=chosen)
        torch.cuda.synchronize()
        assert torch.allclose(out[0].float(), out[1].float(), rtol=2.0 ** -9, atol=2.0 ** -9)


# ---- refusals --------------------------------------------------------------------
def test_refusals(gpu):
    import torch
    _say("paged refusals")
    i32 = dict(dtype=torch.int32, device="cuda")
    g = _bitmap(gpu, np.ones(64, bool))
    n, table = torch.ones(2, **i32), torch.zeros(2, 4, **i32)
    slots = torch.zeros(8, dtype=torch.int64, device="cuda")
    plan = dict(free_pages=g, n_pages=64, page_size=16, d_cached=n, d_new=n, d_table=table, d_slots=slots,
                d_starts=torch.zeros(3, **i32), d_kv_len=torch.zeros(2, **i32), d_taken=torch.zeros(4, **i32),
                d_counts=torch.zeros(3, **i32))
    for what, code in ((dict(page_size=12), gpu.CR_ERR_INVALID), (dict(page_size=0), gpu.CR_ERR_INVALID),
                       (dict(d_slots=slots.int()), gpu.CR_ERR_INVALID), (dict(d_new=n[:1]), gpu.CR_ERR_INVALID),
                       (dict(d_table=table.long()), gpu.CR_ERR_INVALID), (dict(d_table=table.t()), gpu.CR_ERR_INVALID),
                       (dict(d_starts=torch.zeros(2, **i32)), gpu.CR_ERR_INVALID),
                       (dict(d_counts=torch.zeros(3, dtype=torch.int32)), gpu.CR_ERR_INVALID),
                       (dict(n_pages=1 << 28), gpu.CR_ERR_UNSUPPORTED)):
        with pytest.raises(gpu.CrError) as e:
            gpu.paged_plan(**{**plan, **what})
        assert e.value.code == code, what
    h = dict(dtype=torch.float16, device="cuda")
    kc, k = torch.zeros(4, 16, 2, 64, **h), torch.zeros(3, 2, 64, **h)
    for bad in (dict(d_k=k.float()), dict(d_v=k[:2]), dict(d_slots=slots[:2]), dict(d_slots=slots[:3].int()),
                dict(d_k=k[:, :1]), dict(d_v_cache=kc.float()), dict(d_k_cache=kc[:, :12], d_v_cache=kc[:, :12]),
                dict(d_k=k.transpose(1, 2)), dict(d_k=k.cpu())):
        with pytest.raises(gpu.CrError):
            gpu.paged_append(**{**dict(d_k=k, d_v=k, d_slots=slots[:3], d_k_cache=kc, d_v_cache=kc.clone()), **bad})
    sel = dict(visible=g, d_table=table, d_starts=torch.zeros(3, **i32), d_kv_len=n, page_size=16,
               d_sel=torch.zeros(2, 64, **i32), d_sel_len=n.clone(), d_limits=torch.zeros(0, **i32))
    gpu.paged_select(**sel)
    for bad in (dict(d_sel=torch.zeros(2, 63, **i32)), dict(page_size=3), dict(d_sel_len=n[:1]),
                dict(d_sel=torch.zeros(1, 64, **i32)), dict(d_limits=slots)):
        with pytest.raises(gpu.CrError):
            gpu.paged_select(**{**sel, **bad})
    torch.cuda.synchronize()
    gpu.free(g)


def test_allocation_failure_is_reported(gpu):
    import torch
    _say("paged allocation failure")
    i32 = dict(dtype=torch.int32, device="cuda")
    g = _bitmap(gpu, np.ones(64, bool))
    n = torch.ones(2, **i32)
    lib = gpu.load()
    lib.cr_debug_fail_device_allocs(0, 1)
    try:
        with pytest.raises(gpu.CrError) as e:
            gpu.paged_plan(g, 64, 16, n, n, torch.zeros(2, 4, **i32), torch.zeros(2, dtype=torch.int64, device="cuda"),
                           torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros(4, **i32), torch.zeros(3, **i32))
        assert e.value.code == gpu.CR_ERR_ALLOC
    finally:
        lib.cr_debug_fail_device_allocs(0, 0)
    gpu.free(g)


def test_select_with_a_universe_inside_a_page(gpu):
    """Without n_pages, the page that the bitmap's universe ends in is one of them: what the set holds of it is listed."""
    import torch
    _say("select, universe inside a page")
    i32 = dict(dtype=torch.int32, device="cuda")
    for kind in ("bitmap", "stored"):
        visible = np.ones(37, bool)
        visible[[0, 33]] = False
        g = _bitmap(gpu, visible, kind)
        sel, length, limits = torch.full((1, 64), -5, **i32), torch.zeros(1, **i32), torch.zeros(1, **i32)
        table = torch.tensor([[2, 0, 3, 1]], **i32)
        gpu.paged_select(g, table, torch.tensor([0, 1], **i32), torch.tensor([64], **i32), 16, sel, length, limits)
        torch.cuda.synchronize()
        gpu.free(g)
        want = [32, 34, 35, 36] + list(range(1, 32))
        assert int(length) == int(limits) == len(want) and sel[0, :len(want)].tolist() == want
