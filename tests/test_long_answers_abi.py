"""Refusals of the operators for long and speculative answers that need no GPU: each is decided from the host's
arguments, before any device memory is touched."""
import ctypes as C

import pytest

import curoaring as cr

OK, INVALID, UNSUPPORTED = cr.CR_OK, cr.CR_ERR_INVALID, cr.CR_ERR_UNSUPPORTED
P = 0x1000  # stands for a device address: nothing is read from it


def _cache(**kw):
    c = cr.PagedCache(P, P, 16 * 2 * 64, 2 * 64, 64, 16 * 2 * 64, 2 * 64, 64, 8, 16, 2, 64, cr.F16)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _filled(kind, base, bad):
    a = kind()
    for k, v in {**base, **bad}.items():
        setattr(a, k, v)
    return a


ROTARY = dict(q=P, q_token_stride=256, q_head_stride=64, q_out=P, out_token_stride=256, out_head_stride=64, k=P,
              k_token_stride=128, k_head_stride=64, v=P, v_token_stride=128, v_head_stride=64, d_positions=P, d_freqs=P,
              d_slots=P, n_tokens=3, n_heads=4, rotated=64, interleaved=0, magnitude=1.0)


@pytest.mark.parametrize("args,cache,code", [
    (dict(q=None), {}, INVALID), (dict(q_out=None), {}, INVALID), (dict(k=None), {}, INVALID), (dict(v=None), {}, INVALID),
    (dict(d_positions=None), {}, INVALID), (dict(d_freqs=None), {}, INVALID), (dict(d_slots=None), {}, INVALID),
    (dict(rotated=63), {}, INVALID), (dict(rotated=66), {}, INVALID), ({}, dict(page_size=12), INVALID),
    ({}, dict(page_size=0), INVALID), ({}, dict(dtype=3), INVALID), ({}, dict(k=None), INVALID), ({}, dict(v=None), INVALID),
    ({}, dict(head_dim=0), INVALID), (dict(rotated=8192), dict(head_dim=8192), UNSUPPORTED),
    (dict(n_heads=1 << 24), {}, UNSUPPORTED), (dict(n_tokens=1 << 31), {}, UNSUPPORTED), (dict(n_tokens=0, k=None), {}, OK),
    (dict(out_head_stride=0), {}, INVALID), (dict(out_head_stride=63), {}, INVALID), (dict(out_token_stride=0), {}, INVALID)])
def test_rotary(args, cache, code):
    assert cr.load().cr_paged_rotary(C.byref(_filled(cr.PagedRotaryArgs, ROTARY, args)), C.byref(_cache(**cache)), None) == code


WEIGHTS = dict(q=P, q_token_stride=256, q_head_stride=64, lse=P, n_tokens=3, n_heads=4, n_requests=2, d_starts=P, d_kv_len=P,
               d_table=P, table_cols=4, table_stride=4, d_out=P, out_stride=64, scale=0.125, decay=1.0, causal=1)


@pytest.mark.parametrize("args,cache,code", [
    (dict(q=None), {}, INVALID), (dict(lse=None), {}, INVALID), (dict(d_starts=None), {}, INVALID),
    (dict(d_kv_len=None), {}, INVALID), (dict(d_table=None), {}, INVALID), (dict(table_stride=3), {}, INVALID),
    (dict(d_out=None), {}, INVALID), (dict(out_stride=63), {}, INVALID), (dict(d_past=P, past_stride=63), {}, INVALID),
    (dict(n_heads=5), {}, INVALID), (dict(n_heads=0), {}, INVALID), ({}, dict(n_heads=0), INVALID),
    ({}, dict(page_size=24), INVALID), ({}, dict(head_dim=0), INVALID), ({}, dict(k=None), INVALID),
    ({}, dict(dtype=cr.F32), UNSUPPORTED), ({}, dict(head_dim=264), UNSUPPORTED), ({}, dict(head_dim=60), UNSUPPORTED),
    (dict(q=P + 8), {}, UNSUPPORTED), (dict(q_head_stride=68), {}, UNSUPPORTED), ({}, dict(k_slot_stride=132), UNSUPPORTED),
    ({}, dict(n_pages=1 << 28), UNSUPPORTED), (dict(n_tokens=1 << 31), {}, UNSUPPORTED),
    (dict(n_requests=1 << 24), {}, UNSUPPORTED), (dict(n_requests=1 << 22), {}, UNSUPPORTED), (dict(n_tokens=1 << 30), {}, UNSUPPORTED),
    (dict(table_cols=1 << 24, table_stride=1 << 24, out_stride=1 << 28, n_requests=256), {}, UNSUPPORTED),
    (dict(n_requests=0, q=None), {}, OK), (dict(table_cols=0, d_table=None, d_out=None), dict(v=None), OK)])
def test_weights(args, cache, code):
    a = _filled(cr.PagedWeightsArgs, WEIGHTS, args)
    assert cr.load().cr_paged_weights(C.byref(a), C.byref(_cache(**cache)), None) == code


EVICT = dict(d_weights=P, weights_stride=64, d_positions=P, positions_stride=64, d_kept=P, d_seen=P, d_kv_len=P, d_keep=P,
             d_table=P, table_cols=4, table_stride=4, page_size=16, n_pages=8, n_requests=2, sinks=1, recent=2,
             d_weights_out=P, weights_out_stride=64, d_positions_out=P, positions_out_stride=64, d_len=P + 256, d_moves=P,
             moves_cap=32, moves_stride=32, d_n_moves=P + 512, d_freed=P, freed_cap=8, d_counts=P)


@pytest.mark.parametrize("bad,code", [
    (dict(d_weights=None), INVALID), (dict(weights_stride=63), INVALID), (dict(positions_stride=63), INVALID),
    (dict(d_kept=None), INVALID), (dict(d_positions_out=None), INVALID), (dict(d_kv_len=None), INVALID),
    (dict(d_keep=None), INVALID), (dict(d_table=None), INVALID), (dict(table_stride=3), INVALID), (dict(page_size=0), INVALID),
    (dict(page_size=12), INVALID), (dict(d_weights_out=None), INVALID), (dict(weights_out_stride=63), INVALID),
    (dict(positions_out_stride=63), INVALID), (dict(d_len=None), INVALID), (dict(d_moves=None), INVALID),
    (dict(moves_cap=31), INVALID), (dict(moves_stride=31), INVALID), (dict(d_n_moves=None), INVALID),
    (dict(d_freed=None), INVALID), (dict(d_counts=None), INVALID), (dict(n_pages=1 << 28), UNSUPPORTED),
    (dict(n_requests=1 << 20), UNSUPPORTED), (dict(sinks=1 << 31), UNSUPPORTED), (dict(recent=1 << 31), UNSUPPORTED),
    (dict(d_len=P), INVALID), (dict(d_len=P + 4), INVALID), (dict(d_kept=P + 252), INVALID), (dict(d_n_moves=P - 4), INVALID),
    (dict(d_seen=P + 516), INVALID)])
def test_evict(bad, code):
    assert cr.load().cr_paged_evict(C.byref(_filled(cr.PagedEvictArgs, EVICT, bad)), None) == code
    assert b"cr_paged_evict" in cr._lib.cr_last_error()


MOVE = dict(moves=P, cap=32, stride=32, n_moves=P, n=2)


@pytest.mark.parametrize("args,cache,code", [
    (dict(moves=None), {}, INVALID), (dict(stride=31), {}, INVALID), (dict(n_moves=None), {}, INVALID),
    ({}, dict(k=None), INVALID), ({}, dict(v=None), INVALID), ({}, dict(page_size=24), INVALID), ({}, dict(dtype=3), INVALID),
    (dict(cap=1 << 31, stride=1 << 31), {}, UNSUPPORTED), (dict(n=1 << 20), {}, UNSUPPORTED),
    ({}, dict(n_heads=1 << 24), UNSUPPORTED), (dict(n=0, moves=None, n_moves=None), {}, OK), (dict(cap=0, moves=None), {}, OK)])
def test_move(args, cache, code):
    assert cr.load().cr_paged_move(*{**MOVE, **args}.values(), C.byref(_cache(**cache)), None) == code


VERIFY = dict(d_scores=P, row_stride=1000, d_draft=P, draft_row_stride=1000, dtype=cr.F32, n_rows=5, n_requests=2, vocab=1000,
              d_tokens=P, d_starts=P, d_uniform=P, temperature=1.0, d_accepted=P, d_out=P, out_cols=4, out_stride=4)


@pytest.mark.parametrize("bad,code", [
    (dict(d_scores=None), INVALID), (dict(d_scores=P + 2), INVALID), (dict(d_draft=P + 2), INVALID),
    (dict(row_stride=999), INVALID), (dict(draft_row_stride=999), INVALID), (dict(dtype=3), INVALID), (dict(vocab=0), INVALID),
    (dict(d_tokens=None), INVALID), (dict(d_starts=None), INVALID), (dict(d_uniform=None), INVALID),
    (dict(temperature=0.0), INVALID), (dict(temperature=-1.0), INVALID), (dict(temperature=float("nan")), INVALID),
    (dict(temperature=float("inf")), INVALID), (dict(d_accepted=None), INVALID), (dict(d_out=None), INVALID),
    (dict(out_stride=3), INVALID), (dict(allowed=P, d_allowed_bits=P), INVALID),
    (dict(n_rows=1 << 24, vocab=1 << 16, row_stride=1 << 16, draft_row_stride=1 << 16), UNSUPPORTED),
    (dict(n_requests=1 << 20), UNSUPPORTED), (dict(vocab=1 << 31, n_rows=1), UNSUPPORTED),
    (dict(n_requests=0, d_scores=None), OK)])
def test_verify(bad, code):
    assert cr.load().cr_draft_verify(C.byref(_filled(cr.DraftVerifyArgs, VERIFY, bad)), None) == code


def test_nothing_to_point_at():
    lib = cr.load()
    assert lib.cr_paged_rotary(None, None, None) == lib.cr_paged_weights(None, None, None) == INVALID
    assert lib.cr_paged_evict(None, None) == lib.cr_draft_verify(None, None) == lib.cr_paged_move(P, 1, 1, P, 1, None, None) == INVALID


@pytest.mark.parametrize("bad", [dict(rotated=63), dict(rotated=-2), dict(base=0.0), dict(factor=0.0), dict(scaling="half")])
def test_frequencies_refused(bad):
    with pytest.raises(cr.CrError):
        cr.rotary_frequencies(**{**dict(rotated=64, device="cpu"), **bad})


def test_frequencies():
    import math
    plain, one = cr.rotary_frequencies(64, device="cpu")
    assert one == 1.0 and plain.shape == (32,) and all(
        abs(float(f) - 10000.0 ** (-2 * i / 64)) < 1e-15 for i, f in enumerate(plain))
    linear, _ = cr.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert float((linear * 4 - plain).abs().max()) < 1e-15
    base, _ = cr.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert float(base[0]) == 1.0 and abs(float(base[-1] * 4 / plain[-1]) - 1) < 1e-12
    parts, m = cr.rotary_frequencies(64, scaling="parts", factor=4.0, original=4096, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert bool((parts[turns > 32] == plain[turns > 32]).all())
    assert float((parts[turns < 1] * 4 - plain[turns < 1]).abs().max()) < 1e-15
    assert bool((parts <= plain).all()) and bool((parts * 4 >= plain - 1e-15).all()) and abs(m - 1 - 0.1 * math.log(4)) < 1e-15
    assert cr.rotary_frequencies(0, device="cpu")[0].numel() == 0


class _On:
    """A host tensor that says it is on a device; the library is not called with it."""

    def __init__(self, t, device):
        self.t, self.number = t, device

    is_cuda = True

    def get_device(self):
        return self.number

    def __getattr__(self, name):
        return getattr(self.t, name)


def _calls():
    import torch
    i32, half = dict(dtype=torch.int32), dict(dtype=torch.float16)
    k, cache = torch.zeros(2, 2, 64, **half), torch.zeros(4, 16, 2, 64, **half)
    n, starts, table = torch.ones(2, **i32), torch.zeros(3, **i32), torch.zeros(2, 4, **i32)
    f64, rows = torch.zeros(32, dtype=torch.float64), torch.zeros(2, 64)
    return {
        "paged_rotary": (dict(d_k=k, d_v=k, d_positions=n, d_freqs=f64, d_slots=torch.zeros(2, dtype=torch.int64),
                              d_k_cache=cache, d_v_cache=cache, d_q=k, d_q_out=k.clone()), {}),
        "paged_weights": (dict(d_q=k, d_k_cache=cache, d_table=table, d_starts=starts, d_kv_len=n, d_lse=torch.zeros(2, 2),
                               d_out=rows, d_past=rows, d_new=n), {}),
        "paged_evict": (dict(d_weights=rows, d_kv_len=n, d_keep=n, d_table=table, d_weights_out=rows.clone(), d_len=n,
                             d_moves=torch.zeros(2, 32, 2, **i32), d_n_moves=n, d_freed=n, d_counts=n,
                             d_positions=torch.zeros(2, 64, **i32), d_kept=n, d_seen=n,
                             d_positions_out=torch.zeros(2, 64, **i32)), dict(page_size=16)),
        "paged_move": (dict(d_moves=torch.zeros(2, 32, 2, **i32), d_n_moves=n, d_k_cache=cache, d_v_cache=cache), {}),
        "draft_verify": (dict(d_scores=torch.zeros(2, 9), d_tokens=n, d_starts=starts, d_uniform=torch.zeros(2), d_accepted=n,
                              d_out=table, d_draft=torch.zeros(2, 9), allowed=torch.zeros(1, **i32)), {})}


def test_tensors_of_another_device_are_refused(monkeypatch):
    import torch
    called = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: called.append(name) or OK

    monkeypatch.setattr(cr, "load", Library)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 2)
    for here in (0, 1):
        monkeypatch.setattr(cr, "_devices", None)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: here)
        for name, (tensors, rest) in _calls().items():
            on = {x: _On(t, here) for x, t in tensors.items()}
            called.clear()
            getattr(cr, name)(**on, **rest)
            assert called == ["cr_" + name]
            for x, t in tensors.items():
                with pytest.raises(cr.CrError) as e:
                    getattr(cr, name)(**{**on, x: _On(t, 1 - here)}, **rest)
                assert e.value.code == INVALID and "current CUDA device" in str(e.value), (name, x)
            assert len(called) == 1


@pytest.mark.parametrize("name,bad", [
    ("paged_rotary", "d_freqs"), ("paged_rotary", "d_positions"), ("paged_rotary", "d_q"), ("paged_weights", "d_out"),
    ("paged_weights", "d_lse"), ("paged_weights", "d_q"), ("paged_weights", "d_new"), ("paged_evict", "d_moves"),
    ("paged_evict", "d_weights"), ("paged_evict", "d_positions"), ("paged_evict", "d_counts"), ("paged_move", "d_moves"),
    ("draft_verify", "d_draft"), ("draft_verify", "d_uniform"), ("draft_verify", "d_out"), ("draft_verify", "d_scores")])
def test_other_types_and_shapes_are_refused(monkeypatch, name, bad):
    import torch

    class Library:
        def __getattr__(self, name):
            return lambda *a: OK

    monkeypatch.setattr(cr, "load", Library)
    monkeypatch.setattr(cr, "_devices", 1)
    tensors, rest = _calls()[name]
    on = {x: _On(t, 0) for x, t in tensors.items()}
    getattr(cr, name)(**on, **rest)
    for other in (tensors[bad].to(torch.int16), tensors[bad][..., None], tensors[bad].new_zeros(tensors[bad].shape[:-1] + (1, 3))):
        with pytest.raises(cr.CrError) as e:
            getattr(cr, name)(**{**on, bad: _On(other, 0)}, **rest)
        assert e.value.code == INVALID
