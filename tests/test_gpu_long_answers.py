"""The operators for long and speculative answers together: the C++ host API (tests/cpp/long_answers_check.cpp), the
example against the same model computed densely, calls captured into graphs, and failed allocations."""
import importlib.util
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def _say(*a):
    print("CASE", *a, flush=True)


def test_cpp_api():
    exe = os.path.join(ROOT, "tests", "cpp", "long_answers_check")
    assert os.path.exists(exe), "tests/cpp/long_answers_check is built by __graft_entry__.build()"
    _say("cpp long_answers_check")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "long_answers_check: OK" in r.stdout, r.stdout + r.stderr


def _example():
    path = os.path.join(ROOT, "cu-roaring-bitmap_amd", "examples", "speculative.py")
    spec = importlib.util.spec_from_file_location("speculative_example", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _dense(model, tokens):
    """Scores [T, vocab] of a sequence, positions and attention written out in fp32."""
    import torch
    t, half = len(tokens), model.dim // 2
    angle = torch.arange(t, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, device="cuda", dtype=torch.float64) / half)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    see = torch.ones((t, t), dtype=torch.bool, device="cuda").tril()

    def turned(x):
        x = x.float()
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    def attend(layer, q, k, v):
        group = model.heads // model.kv_heads
        q, k, v = turned(q), turned(k).repeat_interleave(group, 1), v.float().repeat_interleave(group, 1)
        x = torch.stack([q[:, h] @ k[:, h].T.contiguous() for h in range(model.heads)]) * model.dim ** -0.5
        p = torch.softmax(x.masked_fill(~see, float("-inf")), -1)
        return torch.stack([p[h] @ v[:, h].contiguous() for h in range(model.heads)], 1).to(model.dtype)

    return model.forward(torch.tensor(tokens, device="cuda"), attend)


@pytest.mark.parametrize("drafts,same", [(4, False), (1, False), (3, True), (0, False)])
def test_answers_are_the_models_own(gpu, drafts, same):
    """At a low temperature every token is one of the model's best, whatever drafts it and however many are accepted.
    Activations are rounded to 11 bits some 20 times on the way to a score of size ~1: 0.05 is several times what adds
    up.  A token 0.2 below the best is drawn once in e^20 times."""
    ex = _example()
    _say("speculative example", drafts, same)
    rng = np.random.default_rng(7)
    model = ex.RotaryDecoder(vocab=500)
    draft = model if same else ex.RotaryDecoder(vocab=500, layers=1)
    prompts = [rng.integers(0, 500, m).tolist() for m in (1, 37, 130)]
    session = ex.Session(model, draft, 3, cols=16, pages=64)
    if same:
        session.caches[draft] = session.caches[model]
    answers, share = ex.generate(session, prompts, None, drafts, 24, temperature=0.01)
    assert share > 0.8 if same else share >= 0
    for p, a in zip(prompts, answers):
        assert len(a) >= 24
        scores = _dense(model, p + a)[len(p) - 1:-1]
        got = scores.gather(1, scores.new_tensor(a).long()[:, None])[:, 0]
        assert (scores.amax(1) - got).max() < 0.25
    assert session.cached.tolist() == [len(p) + len(a) - 1 for p, a in zip(prompts, answers)]
    assert session.seen.tolist() == session.cached.tolist()
    session.close()


def test_a_bounded_cache(gpu):
    """Answers longer than the cache: what is kept, where it lies, and what is free again."""
    import torch
    ex = _example()
    _say("speculative example with eviction")
    rng = np.random.default_rng(8)
    model, draft = ex.RotaryDecoder(vocab=500), ex.RotaryDecoder(vocab=500, layers=1)
    prompts = [rng.integers(0, 500, m).tolist() for m in (5, 90, 150)]
    ids = torch.arange(2, 500, 3, dtype=torch.int32, device="cuda")
    allowed = ex.cr.upload_from_device_ids(ids, 500)
    keep, pages = 64, 48
    session = ex.Session(model, draft, 3, cols=16, pages=pages, keep=keep, sinks=4, recent=16)
    answers, _ = ex.generate(session, prompts, allowed, 4, 100, temperature=1.0, pinned=8)
    session.evict()
    for r, (p, a) in enumerate(zip(prompts, answers)):
        assert np.isin(a, ids.cpu().numpy()).all()
        n, seen = int(session.cached[r]), int(session.seen[r])
        assert seen == len(p) + len(a) - 1 and n == keep
        at = session.positions[r, :n].tolist()
        assert len(set(at)) == n and set(range(seen - 16, seen)) <= set(at)
        assert set(range(min(8, len(p)))) <= set(at)  # pinned, or the first four
        w = session.weights[r, :n]
        assert bool((w >= 0).all()) and bool(torch.isfinite(w).all())
    held = sum(-(-int(n) // 16) for n in session.cached)
    assert ex.cr.cardinality(session.free) == pages - held
    assert ex.cr.cardinality(session.pinned) == 21
    ex.cr.free(allowed)
    session.close()


def _step(gpu, seed, requests=3, kv=700):
    """The calls of a step on state of its own: (name, call(stream), outputs)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    i32 = dict(dtype=torch.int32, device="cuda")
    page, heads, kv_heads, dim, rows = 16, 4, 2, 64, 4
    cols = -(-(kv + rows) // page)
    pages = requests * cols
    half = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).view(requests, cols)
    starts, kv_len = torch.arange(0, rows * requests + 1, rows, **i32), torch.full((requests,), kv, **i32)
    q, k, v = half(rows * requests, heads, dim), half(rows * requests, kv_heads, dim), half(rows * requests, kv_heads, dim)
    kc, vc = half(pages, page, kv_heads, dim), half(pages, page, kv_heads, dim)
    at = (kv - rows + torch.arange(rows, device="cuda")).repeat(requests)
    row = torch.arange(requests, device="cuda").repeat_interleave(rows)
    slots = table.long()[row, at // page] * page + at % page
    q_out, out, lse = torch.empty_like(q), torch.empty_like(q), torch.zeros(rows * requests, heads, device="cuda")
    room = cols * page
    weights, w_out = torch.zeros(requests, room, device="cuda"), torch.zeros(requests, room, device="cuda")
    past = torch.rand(requests, room, device="cuda", generator=g)
    length, n_moves, counts = torch.zeros(requests, **i32), torch.zeros(requests, **i32), torch.zeros(2, **i32)
    moves, freed = torch.zeros(requests, room // 2, 2, **i32), torch.zeros(pages, **i32)
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    x, y = torch.randn(rows * requests, 5003, device="cuda", generator=g), torch.randn(rows * requests, 5003, device="cuda", generator=g)
    tokens = y.argmax(1).roll(1).to(torch.int32)
    u = torch.rand(rows * requests, device="cuda", generator=g)
    accepted, drawn = torch.zeros(requests, **i32), torch.zeros(requests, rows, **i32)
    sparse = gpu.upload_from_ids(np.arange(0, pages * page, 7, dtype=np.uint32), pages * page, gpu.PROMOTE_KEEP_DEFAULT)
    allowed = gpu.upload_from_ids(np.arange(0, 5003, 5, dtype=np.uint32), 5003, gpu.PROMOTE_KEEP_DEFAULT)
    freqs, _ = gpu.rotary_frequencies(dim)
    keep = torch.full((requests,), kv // 2, **i32)

    def evict(s):
        gpu.paged_evict(weights, kv_len, keep, table, page, w_out, length, moves, n_moves, freed, counts, recent=5,
                        pinned=sparse, n_pages=pages, stream=s)
        k2.copy_(kc)
        v2.copy_(vc)
        gpu.paged_move(moves, n_moves, k2, v2, stream=s)

    return [
        ("rotary", lambda s: gpu.paged_rotary(k, v, at.to(torch.int32), freqs, slots, kc, vc, d_q=q, d_q_out=q_out, stream=s),
         (q_out, kc, vc)),
        ("attention", lambda s: gpu.paged_attention(q_out, kc, vc, table, starts, kv_len, out, d_lse=lse, stream=s), (out, lse)),
        ("weights", lambda s: gpu.paged_weights(q_out, kc, table, starts, kv_len, lse, weights, d_past=past, visible=sparse,
                                                stream=s), (weights,)),
        ("evict", evict, (w_out, length, n_moves, moves, freed, counts, k2, v2)),
        ("verify", lambda s: gpu.draft_verify(x, tokens, starts, u, accepted, drawn, d_draft=y, allowed=allowed, stream=s),
         (accepted, drawn)),
        ("verify looked up", lambda s: gpu.draft_verify(x, tokens, starts, u, accepted, drawn, stream=s), (accepted, drawn)),
    ], (sparse, allowed), (x, y, past, u)


@pytest.mark.parametrize("which", range(6))
def test_captured_calls(gpu, which):
    """Two graphs of a call captured on one stream, each replayed several times on new inputs, with eager calls of the
    same operator on that stream between them: every replay gives what the eager call gives.  Then both at once, on
    streams of their own: neither has the other's workspace."""
    import torch
    steps = [_step(gpu, seed) for seed in (1, 2)]
    name = steps[0][0][which][0]
    _say("captured", name)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for calls, _, _ in steps:
            for _, call, _ in calls[:which + 1]:
                call(side)
    side.synchronize()
    graphs = []
    for calls, _, _ in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls[which][1](side)
        graphs.append(graph)
    for turn in range(4):
        for (calls, _, inputs), graph in zip(steps, graphs):
            with torch.cuda.stream(side):
                for t in inputs:
                    t.mul_(1.0 - 0.125 * turn)
                for _, call, _ in calls[:which + 1]:
                    call(side)
                want = [t.clone() for t in calls[which][2]]
                for t in calls[which][2]:
                    if name not in ("rotary",):
                        t.zero_()
                graph.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, calls[which][2])), (name, turn)
    wants = [[t.clone() for t in calls[which][2]] for calls, _, _ in steps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (calls, _, _), want in zip(steps, wants):
        assert all(torch.equal(a, b) for a, b in zip(want, calls[which][2])), name
    del graphs, graph
    for _, bitmaps, _ in steps:
        for g in bitmaps:
            gpu.free(g)


def test_allocation_failures_are_reported(gpu):
    """Calls without memory for their workspace: an error, nothing written, and the same call goes through afterwards."""
    import torch
    calls, bitmaps, _ = _step(gpu, 3)
    lib = gpu.load()
    for _, call, _ in calls[:2]:
        call(None)
    for name, call, outputs in calls[2:]:
        _say("allocation failure", name)
        torch.cuda.synchronize()
        gpu.load().cr_mempool_trim(-1, 0)
        before = [t.clone() for t in outputs]
        lib.cr_debug_fail_device_allocs(0, 1)
        try:
            with pytest.raises(gpu.CrError) as e:
                call(None)
            assert e.value.code == gpu.CR_ERR_ALLOC
        finally:
            lib.cr_debug_fail_device_allocs(0, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, outputs)), name
        call(None)
        torch.cuda.synchronize()
        for t in outputs:
            t.zero_() if name == "verify" else None
    for g in bitmaps:
        gpu.free(g)


def test_two_streams_at_once(gpu):
    """The same operators on two streams side by side give what they give alone."""
    import torch
    _say("two streams")
    steps = [_step(gpu, seed, kv=3000) for seed in (4, 5)]
    wants = []
    for calls, _, _ in steps:
        for _, call, _ in calls:
            call(None)
        torch.cuda.synchronize()
        wants.append([[t.clone() for t in outputs] for _, _, outputs in calls])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (calls, _, _), s in zip(steps, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _, call, _ in calls:
                    call(s)
    torch.cuda.synchronize()
    for (calls, bitmaps, _), want in zip(steps, wants):
        for (name, _, outputs), w in zip(calls[:-1], want[:-1]):
            if name != "verify":  # whose outputs the last call wrote over
                assert all(torch.equal(a, b) for a, b in zip(w, outputs)), name
        assert all(torch.equal(a, b) for a, b in zip(want[-1], calls[-1][2]))
        for g in bitmaps:
            gpu.free(g)
