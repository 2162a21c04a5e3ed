"""Refusals of the serving operators that need no GPU: each is decided from the
host's arguments, before any device memory is touched."""
import ctypes as C

import pytest

import curoaring as cr

OK, INVALID, UNSUPPORTED = cr.CR_OK, cr.CR_ERR_INVALID, cr.CR_ERR_UNSUPPORTED
P = 0x1000  # stands for a device address: nothing is read from it


def _bitmap():
    return C.byref(cr.GpuRoaring(universe_size=1024))


def _cache(**kw):
    c = cr.PagedCache(P, P, 16 * 2 * 64, 2 * 64, 64, 16 * 2 * 64, 2 * 64, 64, 8, 16, 2, 64, cr.F16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


PLAN = dict(free=None, n_pages=64, page=16, cached=P, new=P, n=2, table=P, cols=4, stride=4, slots=P, slots_cap=8,
            starts=P, kv=P, taken=P, taken_cap=8, counts=P)


@pytest.mark.parametrize("bad,code", [
    (dict(free=0), INVALID), (dict(page=0), INVALID), (dict(page=12), INVALID), (dict(starts=None), INVALID),
    (dict(counts=None), INVALID), (dict(cached=None), INVALID), (dict(new=None), INVALID), (dict(kv=None), INVALID),
    (dict(table=None), INVALID), (dict(stride=3), INVALID), (dict(slots=None), INVALID), (dict(taken=None), INVALID),
    (dict(n_pages=1 << 28), UNSUPPORTED), (dict(slots_cap=1 << 31), UNSUPPORTED), (dict(n=1 << 24), UNSUPPORTED)])
def test_plan(bad, code):
    a = {**PLAN, **bad}
    a["free"] = None if a["free"] == 0 else _bitmap()
    assert cr.load().cr_paged_plan(*a.values(), None) == code
    assert b"cr_paged_plan" in cr._lib.cr_last_error()


@pytest.mark.parametrize("args,cache,code", [
    (dict(k=None), {}, INVALID), (dict(v=None), {}, INVALID), (dict(slots=None), {}, INVALID),
    ({}, dict(k=None), INVALID), ({}, dict(page_size=24), INVALID), ({}, dict(dtype=3), INVALID),
    (dict(n=(1 << 32) - 1), dict(n_heads=64), UNSUPPORTED), (dict(n=0, k=None), {}, OK)])
def test_append(args, cache, code):
    a = {**dict(k=P, v=P, kt=128, kh=64, vt=128, vh=64, n=3, slots=P), **args}
    assert cr.load().cr_paged_append(*a.values(), C.byref(_cache(**cache)), None) == code


SELECT = dict(visible=1, n_pages=64, page=16, table=P, cols=4, stride=4, starts=P, kv=P, n=2, n_tokens=2, sel=P,
              sel_stride=64, sel_len=P, limits=P)


@pytest.mark.parametrize("bad,code", [
    (dict(visible=0), INVALID), (dict(page=3), INVALID), (dict(table=None), INVALID), (dict(stride=2), INVALID),
    (dict(starts=None), INVALID), (dict(kv=None), INVALID), (dict(sel=None), INVALID), (dict(sel_stride=63), INVALID),
    (dict(sel_len=None), INVALID), (dict(limits=None), INVALID), (dict(n_pages=1 << 28), UNSUPPORTED),
    (dict(n=1 << 31), UNSUPPORTED), (dict(n_tokens=1 << 31), UNSUPPORTED), (dict(n=0, sel=None), OK)])
def test_select(bad, code):
    a = {**SELECT, **bad}
    a["visible"] = _bitmap() if a["visible"] else None
    assert cr.load().cr_paged_select(*a.values(), None) == code


def _attention(**kw):
    a = cr.PagedAttentionArgs(P, 4 * 64, 64, P, 4 * 64, 64, None, 3, 4, 2, P, P, P, 4, 4, None, 0, None, None, 0.125, 1,
                              0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("args,cache,code", [
    (dict(q=None), {}, INVALID), (dict(out=None), {}, INVALID), (dict(d_starts=None), {}, INVALID),
    (dict(d_kv_len=None), {}, INVALID), (dict(d_table=None), {}, INVALID), (dict(table_stride=3), {}, INVALID),
    (dict(n_heads=5), {}, INVALID), ({}, dict(n_heads=0), INVALID), ({}, dict(page_size=12), INVALID),
    ({}, dict(head_dim=0), INVALID), ({}, dict(v=None), INVALID),
    (dict(d_sel=P, sel_stride=63, d_sel_len=P, d_limits=P), {}, INVALID),
    (dict(d_sel=P, sel_stride=64, d_sel_len=None, d_limits=P), {}, INVALID),
    (dict(d_sel=P, sel_stride=64, d_sel_len=P, d_limits=None), {}, INVALID),
    ({}, dict(dtype=cr.F32), UNSUPPORTED), ({}, dict(head_dim=264), UNSUPPORTED), ({}, dict(head_dim=60), UNSUPPORTED),
    (dict(q=P + 8), {}, UNSUPPORTED), (dict(q_head_stride=68), {}, UNSUPPORTED), ({}, dict(v_slot_stride=132), UNSUPPORTED),
    ({}, dict(n_pages=1 << 28), UNSUPPORTED), (dict(n_tokens=1 << 31), {}, UNSUPPORTED),
    (dict(n_requests=1 << 24), {}, UNSUPPORTED), (dict(n_tokens=1 << 29, n_heads=64), {}, UNSUPPORTED),
    (dict(n_tokens=0, q=None), {}, OK)])
def test_attention(args, cache, code):
    assert cr.load().cr_paged_attention(C.byref(_attention(**args)), C.byref(_cache(**cache)), None) == code


BEAM = dict(x=P, dtype=cr.F32, batch=2, beams=3, vocab=100, batch_stride=300, beam_stride=100, cum=P, lse=None,
            allowed=None, bits=None, bits_stride=0, k=4, scores=P, tokens=P, parents=P)


@pytest.mark.parametrize("bad,code", [
    (dict(x=None), INVALID), (dict(x=P + 2), INVALID), (dict(dtype=3), INVALID), (dict(beams=0), INVALID),
    (dict(vocab=0), INVALID), (dict(beam_stride=99), INVALID), (dict(cum=None), INVALID), (dict(allowed=1, bits=P), INVALID),
    (dict(scores=None), INVALID), (dict(tokens=None), INVALID), (dict(parents=None), INVALID),
    (dict(k=257), UNSUPPORTED), (dict(vocab=1 << 30, beam_stride=1 << 30), UNSUPPORTED), (dict(batch=1 << 20), UNSUPPORTED),
    (dict(batch=0, x=None), OK), (dict(k=0, x=None), OK)])
def test_beam_select(bad, code):
    a = {**BEAM, **bad}
    a["allowed"] = _bitmap() if a["allowed"] else None
    assert cr.load().cr_beam_select(*a.values(), None) == code


REORDER = dict(src=P, parents=P, batch=2, w=3, k=4, row=64, src_stride=64, dst_stride=64, len=None, unit=0, dst=2 * P)


@pytest.mark.parametrize("bad,code", [
    (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(parents=None), INVALID), (dict(w=0), INVALID),
    (dict(src_stride=63), INVALID), (dict(dst_stride=63), INVALID), (dict(len=P), INVALID), (dict(dst=P + 64), INVALID),
    (dict(k=65536), UNSUPPORTED), (dict(batch=1 << 30), UNSUPPORTED), (dict(batch=0, src=None), OK),
    (dict(row=0, src=None), OK)])
def test_beam_reorder(bad, code):
    assert cr.load().cr_beam_reorder(*{**REORDER, **bad}.values(), None) == code


def test_tensors_on_the_host_are_refused():
    import torch
    i32, k = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.float16)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    for call in (lambda: cr.paged_plan(cr.GpuRoaring(), 8, 16, i32, i32, torch.zeros(2, 4, dtype=torch.int32),
                                       torch.zeros(8, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), i32, i32,
                                       torch.zeros(3, dtype=torch.int32)),
                 lambda: cr.paged_append(k, k, torch.zeros(2, dtype=torch.int64), cache, cache),
                 lambda: cr.paged_attention(k, cache, cache, torch.zeros(2, 4, dtype=torch.int32),
                                            torch.zeros(3, dtype=torch.int32), i32, k),
                 lambda: cr.beam_select(torch.zeros(1, 2, 10), torch.zeros(1, 2), torch.zeros(1, 3),
                                        torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32)),
                 lambda: cr.beam_reorder(k, torch.zeros(2, 2, dtype=torch.int32), k.clone())):
        with pytest.raises(cr.CrError) as e:
            call()
        assert e.value.code == INVALID


class _On:
    """A host tensor that says it is on a device; the library is not called with it."""

    def __init__(self, t, device):
        self.t, self.number = t, device

    is_cuda = True

    def get_device(self):
        return self.number

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_tensors_of_another_device_are_refused(monkeypatch):
    import torch
    i32, half = dict(dtype=torch.int32), dict(dtype=torch.float16)
    k, cache = torch.zeros(2, 2, 64, **half), torch.zeros(4, 16, 2, 64, **half)
    n, starts, table = torch.ones(2, **i32), torch.zeros(3, **i32), torch.zeros(2, 4, **i32)
    calls = {
        "paged_plan": (dict(d_cached=n, d_new=n, d_table=table, d_slots=torch.zeros(8, dtype=torch.int64), d_starts=starts,
                            d_kv_len=n, d_taken=n, d_counts=starts), dict(free_pages=cr.GpuRoaring(), n_pages=8, page_size=16)),
        "paged_append": (dict(d_k=k, d_v=k, d_slots=torch.zeros(2, dtype=torch.int64), d_k_cache=cache, d_v_cache=cache), {}),
        "paged_select": (dict(d_table=table, d_starts=starts, d_kv_len=n, d_sel=torch.zeros(2, 64, **i32), d_sel_len=n,
                              d_limits=n), dict(visible=cr.GpuRoaring(), page_size=16)),
        "paged_attention": (dict(d_q=k, d_k_cache=cache, d_v_cache=cache, d_table=table, d_starts=starts, d_kv_len=n, d_out=k,
                                 d_lse=torch.zeros(2, 2)), {}),
        "beam_select": (dict(d_scores=torch.zeros(1, 2, 10), d_cum=torch.zeros(1, 2), d_out_scores=torch.zeros(1, 3),
                             d_out_tokens=torch.zeros(1, 3, **i32), d_out_parents=torch.zeros(1, 3, **i32),
                             d_lse=torch.zeros(1, 2), allowed=torch.zeros(1, **i32)), {}),
        "beam_reorder": (dict(d_src=k, d_parents=torch.zeros(2, 2, **i32), d_dst=k.clone(), d_len=torch.ones(2, 2, **i32)), {})}
    called = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: called.append(name) or OK

    monkeypatch.setattr(cr, "load", Library)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 2)
    for here in (0, 1):
        monkeypatch.setattr(cr, "_devices", None)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: here)
        for name, (tensors, rest) in calls.items():
            on = {x: _On(t, here) for x, t in tensors.items()}
            called.clear()
            getattr(cr, name)(**on, **rest)
            assert called == ["cr_" + name]
            for x, t in tensors.items():
                with pytest.raises(cr.CrError) as e:
                    getattr(cr, name)(**{**on, x: _On(t, 1 - here)}, **rest)
                assert e.value.code == INVALID and "current CUDA device" in str(e.value), (name, x)
            assert len(called) == 1
