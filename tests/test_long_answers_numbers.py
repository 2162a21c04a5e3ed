"""Numbers that the Python calls for long and speculative answers cannot pass on are refused as the library refuses."""
import pytest

import curoaring as cr
from test_long_answers_abi import OK, _calls, _On


@pytest.mark.parametrize("bad", [dict(page_size=0), dict(page_size=-16), dict(page_size=1 << 32), dict(n_pages=-1),
                                 dict(n_pages=1 << 32), dict(sinks=-1), dict(recent=1 << 32)])
def test_evict(monkeypatch, bad):
    class Library:
        def __getattr__(self, name):
            return lambda *a: OK

    monkeypatch.setattr(cr, "load", Library)
    monkeypatch.setattr(cr, "_devices", 1)
    tensors, rest = _calls()["paged_evict"]
    on = {x: _On(t, 0) for x, t in tensors.items()}
    cr.paged_evict(**on, **rest)
    with pytest.raises(cr.CrError) as e:
        cr.paged_evict(**on, **{**rest, **bad})
    assert e.value.code == cr.CR_ERR_INVALID
