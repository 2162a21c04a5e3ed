"""The operators for long and speculative answers where their arguments meet: sets that are narrower than what they are
asked about."""
import numpy as np
import pytest

import test_gpu_verify

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
