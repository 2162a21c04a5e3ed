"""draft_verify against the rule in 64 bits, token by token.  A random number that lies within 1e-11 of what it is
compared with says nothing of either side and is drawn anew by the test."""
import numpy as np
import pytest

import orc  # noqa: F401

pytestmark = pytest.mark.gpu

NEAR = 1e-11


def _say(*a):
    print("CASE", *a, flush=True)


def shares(x, temperature, allowed):
    x = np.where(np.isnan(x) | ~allowed, -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros(x.size)
    if top == np.inf:
        e = (x == np.inf).astype(np.float64)
    else:
        e = np.exp((x - top) / temperature)
    return e / e.sum()


def verify_oracle(x, draft, tokens, uniform, temperature, allowed):
    """Of one request's rows: (accepted, the token behind, how near a random number came to its border)."""
    n, v = x.shape
    near = np.inf
    for j in range(n):
        p = shares(x[j], temperature, allowed[j])
        if j == n - 1:
            rest = p
            break
        d = int(tokens[j + 1])
        there = 0 <= d < v
        if draft is None:
            q = np.zeros(v)
            if there:
                q[d] = 1.0
        else:
            q = shares(draft[j], temperature, allowed[j])
        pd, qd = (p[d], q[d]) if there else (0.0, 1.0)
        near = min(near, abs(float(uniform[j]) * qd - pd) if pd > 0 else np.inf)
        if float(uniform[j]) * qd < pd:
            continue
        rest = np.maximum(p - q, 0.0)
        if rest.sum() <= 1e-14:
            rest = p
        break
    if rest.sum() == 0:
        return j, -1, near
    upto, mark = np.cumsum(rest), float(uniform[n - 1]) * rest.sum()
    near = min(near, np.abs(upto[rest > 0] - mark)[:-1].min(initial=np.inf))
    over = np.nonzero((rest > 0) & (upto > mark))[0]
    return j, int(over[0]) if over.size else int(np.nonzero(rest > 0)[0][-1]), near


class Problem:
    def __init__(self, rows, vocab, dtype="float32", seed=0, temperature=1.0, density=None, kind=None, draft=True, spread=2.5,
                 noise=0.5, pad=0, peak=None):
        import torch
        self.torch, self.rows, self.vocab, self.temperature, self.kind = torch, list(rows), vocab, temperature, kind
        dt, total = getattr(torch, dtype), sum(rows)
        rng = np.random.default_rng(seed)
        x = rng.standard_normal((total, vocab + pad)) * spread
        y = x + rng.standard_normal((total, vocab + pad)) * noise
        if peak is not None:
            x[:, peak] += 60
        cuda = lambda a: torch.from_numpy(a.astype(np.float32)).cuda().to(dt)  # noqa: E731
        self.x, self.draft = cuda(x)[:, :vocab], cuda(y)[:, :vocab] if draft else None
        if kind == "rows":
            self.allowed = rng.random((total, vocab)) < density
        elif density is not None:
            self.allowed = np.repeat(rng.random((1, vocab)) < density, total, 0)
        else:
            self.allowed = np.ones((total, vocab), bool)
        # drawn from the drafting model, as they come
        z = np.where(self.allowed, y[:, :vocab] / temperature + rng.gumbel(size=(total, vocab)), -np.inf)
        self.tokens = np.concatenate([[0], z.argmax(1)[:-1]]).astype(np.int32) if total else np.zeros(0, np.int32)
        self.uniform = rng.random(total).astype(np.float32)
        self.rng = rng

    def run(self, gpu, most=None, stream=None):
        torch, n = self.torch, len(self.rows)
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        most = max(self.rows, default=1) if most is None else most
        allowed = None
        words = lambda m: np.packbits(np.pad(m, ((0, 0), (0, -m.shape[1] % 32))), axis=1, bitorder="little").view(np.int32)  # noqa: E731
        if self.kind in ("bitmap", "arrays"):
            allowed = gpu.upload_from_ids(np.nonzero(self.allowed[0])[0].astype(np.uint32), self.vocab,
                                          gpu.PROMOTE_ALL if self.kind == "bitmap" else gpu.PROMOTE_KEEP_DEFAULT)
        elif self.kind == "rows":
            allowed = cuda(words(self.allowed))
        elif self.kind == "flat":
            allowed = cuda(words(self.allowed[:1]))[0]
        i32 = dict(dtype=torch.int32, device="cuda")
        starts = torch.tensor(np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)).cuda()
        accepted, out = torch.full((n,), -9, **i32), torch.full((n, most + 2), -9, **i32)
        gpu.draft_verify(self.x, cuda(self.tokens), starts, cuda(self.uniform), accepted, out[:, :most], d_draft=self.draft,
                         temperature=self.temperature, allowed=allowed, stream=stream)
        torch.cuda.synchronize()
        if self.kind in ("bitmap", "arrays"):
            gpu.free(allowed)
        assert torch.all(out[:, most:] == -9)
        return accepted.cpu().numpy(), out[:, :most].cpu().numpy()

    def want(self):
        x = self.x.double().cpu().numpy()
        y = None if self.draft is None else self.draft.double().cpu().numpy()
        at, got = 0, []
        for n in self.rows:
            s = slice(at, at + n)
            while n:
                a, t, near = verify_oracle(x[s], None if y is None else y[s], self.tokens[s], self.uniform[s],
                                           np.float64(np.float32(self.temperature)), self.allowed[s])
                if near > NEAR:
                    break
                self.uniform[s] = self.rng.random(n).astype(np.float32)
            got.append((0, [-1]) if n == 0 else (a, [int(v) for v in self.tokens[at + 1:at + 1 + a]] + [t]))
            at += n
        return got

    def check(self, gpu, most=None, **kw):
        want = self.want()
        accepted, out = self.run(gpu, most, **kw)
        for r, (a, tokens) in enumerate(want):
            row = (tokens + [-1] * out.shape[1])[:out.shape[1]]
            assert int(accepted[r]) == a and out[r].tolist() == row, (r, int(accepted[r]), a, out[r].tolist(), row)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [([1], 1), ([5], 7), ([3, 1, 4], 63), ([2] * 40, 500), ([5, 9, 1, 2], 2048),
                                        ([4, 4], 2049), ([3, 6], 10007), ([5], 100003)])
def test_verify(gpu, rows, vocab, dtype, draft):
    _say("verify", rows[:4], vocab, dtype, draft)
    for seed in range(3):
        Problem(rows, vocab, dtype, seed=seed, draft=draft).check(gpu)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("noise", [0.5, 0.01])
@pytest.mark.parametrize("rows", [[9] * 4, [10] * 4, [40], [33] + [1] * 9, [1, 25, 1, 0, 3, 2], [64, 65, 66], [14, 0, 14, 0, 14]])
def test_verify_many_rows(gpu, rows, noise, draft):
    """Requests whose rows are decided by a launch of their own, and long ones among short ones, which are not."""
    _say("verify many rows", rows[:4], noise, draft)
    for vocab in (37, 4099):
        Problem(rows, vocab, "bfloat16", seed=len(rows), noise=noise, draft=draft).check(gpu)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows,vocab", [([3, 2], 131072), ([3, 2], 140001), ([12], 140001), ([2], 300007)])
def test_verify_long_rows(gpu, rows, vocab, draft):
    """More pieces of a row than a wave has lanes."""
    _say("verify long rows", rows, vocab, draft)
    Problem(rows, vocab, "float16", seed=21, draft=draft).check(gpu)
    Problem(rows, vocab, "float16", seed=22, draft=draft, density=0.3, kind="bitmap").check(gpu)


@pytest.mark.parametrize("kind", ["bitmap", "arrays", "flat", "rows"])
@pytest.mark.parametrize("density", [0.0, 0.01, 0.3, 1.0])
def test_verify_allowed(gpu, kind, density):
    _say("verify allowed", kind, density)
    for draft in (True, False):
        Problem([4, 1, 6, 3], 70001, "bfloat16", seed=4, density=density, kind=kind, draft=draft).check(gpu)
        Problem([4, 1, 6, 3] * 5, 301, "float32", seed=5, density=density, kind=kind, draft=draft).check(gpu)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 3.0, 1e-30, 1e30])
def test_verify_temperatures(gpu, temperature):
    _say("verify temperature", temperature)
    for draft in (True, False):
        Problem([4, 3, 5] * 4, 3001, "float32", seed=6, temperature=temperature, draft=draft).check(gpu)


@pytest.mark.parametrize("kind", ["bitmap", "arrays", "flat", "rows"])
@pytest.mark.parametrize("count", [0, 1, 511, 512, 513, 2047, 2048])
def test_allowed_tokens_of_a_piece(gpu, kind, count):
    """So many of every 2048 tokens, in one run or scattered."""
    _say("verify allowed of 2048", kind, count)
    for draft in (True, False):
        for scattered in (True, False):
            p = Problem([4, 1, 6], 7000, "bfloat16", seed=23, density=0.5, kind=kind, draft=draft)
            for rows in (p.allowed if kind == "rows" else p.allowed[:1]):
                rows[:] = False
                for first in range(0, 7000, 2048):
                    n = min(2048, 7000 - first)
                    rows[first + (p.rng.permutation(n)[:count] if scattered else np.arange(n)[max(0, n - count):])] = True
            if kind != "rows":
                p.allowed[:] = p.allowed[:1]
            p.check(gpu)


def test_verify_strides(gpu):
    """Rows that lie apart and begin anywhere."""
    _say("verify strides")
    for pad in (1, 3, 8):
        Problem([4, 3, 5], 5001, "bfloat16", seed=7, pad=pad).check(gpu)
        Problem([4, 3, 5], 5001, "float32", seed=7, pad=pad).check(gpu)


def test_the_same_model_accepts_everything(gpu):
    _say("verify against itself")
    p = Problem([6] * 20, 4001, "float16", seed=8, noise=0.0)
    p.draft = p.x.clone()
    accepted, out = p.run(gpu)
    assert np.all(accepted == 5)
    p.check(gpu)


def test_drafts_that_can_not_be(gpu):
    """Tokens outside the vocabulary, or not allowed, are never accepted."""
    _say("verify impossible drafts")
    for draft in (True, False):
        for bad in (-1, -2 ** 31, 1000, 2 ** 31 - 1):
            p = Problem([4] * 6, 1000, seed=9, draft=draft, noise=0.0)
            p.uniform[:] *= 0.5
            p.tokens[2::4] = bad
            p.check(gpu)
        p = Problem([4] * 6, 1000, seed=9, draft=draft, density=0.5, kind="flat")
        p.tokens[1:] = np.nonzero(~p.allowed[0])[0][:23]
        accepted, out = p.run(gpu)
        assert np.all(accepted == 0) and np.all(p.allowed[0][out[:, 0]])
        p.check(gpu)


def test_rows_without_a_candidate_and_odd_scores(gpu):
    _say("verify odd scores")
    for draft in (True, False):
        p = Problem([3] * 8, 900, seed=10, draft=draft)
        nan, inf = float("nan"), float("inf")
        p.x[0] = -inf
        p.x[4] = nan
        p.x[6, 100:] = nan
        p.x[9, 7:20] = inf
        p.x[12, 3] = inf
        p.x[15, ::2] = -inf
        if draft:
            p.draft[3] = -inf
            p.draft[9, 9:12] = inf
            p.draft[18, ::3] = nan
        p.check(gpu)
        accepted, out = p.run(gpu)
        assert accepted[0] == 0 and out[0].tolist() == [-1, -1, -1]


@pytest.mark.parametrize("u", [0.0, -1.0, 1.0, 2.0, float("nan"), float("inf")])
def test_random_numbers_at_the_ends(gpu, u):
    """0 takes the first token that there is; 1 and more the last one, where rounding does not matter: it may be drawn."""
    _say("verify at", u)
    for draft in (True, False):
        p = Problem([3] * 6, 3000, seed=11, draft=draft, density=0.5, kind="flat")
        p.uniform[:] = u
        accepted, out = p.run(gpu)
        can = np.nonzero(p.allowed[0])[0]
        for r in range(6):
            token = out[r, accepted[r]]
            assert token in can
            if u <= 0:
                assert accepted[r] == 2 and token == can[0]
            elif accepted[r] == 0 and not draft:
                left = [t for t in can if t != p.tokens[3 * r + 1]]
                assert token == left[-1]
        if u <= 0:
            p.check(gpu)


def test_one_token_takes_everything(gpu):
    """The drafted token has all but nothing of p: what is left is drawn from as well as can be."""
    _say("verify one peak")
    p = Problem([3] * 10, 5000, seed=12, draft=False, peak=1234)
    p.tokens[:] = 1234
    accepted, out = p.run(gpu)
    assert np.all(accepted == 2) and np.all(out[:, :2] == 1234)
    p.uniform[:] = 1.0
    accepted, out = p.run(gpu)
    assert np.all(out[np.arange(10), accepted] >= 0)


def test_short_rows_of_output(gpu):
    _say("verify with few columns")
    for most in (0, 1, 2, 9):
        Problem([4, 1, 6], 500, seed=13, noise=0.0).check(gpu, most)


def test_requests_without_rows(gpu):
    _say("verify without rows")
    Problem([0, 3, 0, 0, 2, 0], 500, seed=14).check(gpu)
    Problem([0, 0], 500, seed=14, draft=False).check(gpu, 3)


def test_senseless_device_data_stays_inside(gpu):
    import torch
    _say("verify noise")
    p = Problem([3, 2, 4], 700, seed=15)
    g = torch.Generator(device="cuda").manual_seed(1)
    noise = lambda n: torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=g, device="cuda").to(torch.int32)  # noqa: E731
    for i in range(20):
        accepted, out = torch.full((5,), -9, dtype=torch.int32, device="cuda"), torch.full((5, 6), -9, dtype=torch.int32, device="cuda")
        gpu.draft_verify(p.x, noise(9), noise(4), torch.rand(9, device="cuda"), accepted[1:4], out[1:4], d_draft=p.draft)
        torch.cuda.synchronize()
        assert torch.all(out[0] == -9) and torch.all(out[4] == -9) and accepted[0] == -9 and accepted[4] == -9


def test_tokens_follow_the_model(gpu):
    """Over many random numbers the first token comes as often as p says, whatever was drafted.  40000 draws: a token of
    share p is off by more than 5 sqrt(p (1 - p) / 40000) once in 1.7 million."""
    import torch
    _say("verify frequencies")
    n, v = 40000, 12
    rng = np.random.default_rng(16)
    x, y = rng.standard_normal((2, v)).astype(np.float32)
    p, q = (np.exp(t) / np.exp(t).sum() for t in (x.astype(np.float64), y.astype(np.float64)))
    tokens = np.zeros(2 * n, np.int32)
    tokens[1::2] = rng.choice(v, n, p=q)
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    i32 = dict(dtype=torch.int32, device="cuda")
    accepted, out = torch.zeros(n, **i32), torch.zeros(n, 2, **i32)
    for draft in (cuda(np.tile(y, (2 * n, 1))), None):
        gpu.draft_verify(cuda(np.tile(x, (2 * n, 1))), cuda(tokens), cuda(np.arange(0, 2 * n + 1, 2).astype(np.int32)),
                         cuda(rng.random(2 * n).astype(np.float32)), accepted, out, d_draft=draft)
        torch.cuda.synchronize()
        share = np.bincount(out[:, 0].cpu().numpy(), minlength=v) / n
        assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)), (share, p)


def test_another_stream(gpu):
    import torch
    _say("verify on another stream")
    p = Problem([4, 3, 5], 5001, "bfloat16", seed=17, density=0.3, kind="arrays")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p.check(gpu, stream=s)
