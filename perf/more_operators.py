"""The library's operators for long and speculative answers, as measurable cases.

A server that answers at length rotates queries and keys by their positions,
lets a small model draft tokens that the large one checks, and keeps of a long
context the tokens that attention looks at.  A case is a dict of plain values;
`op` says which operator one pass runs:

  rotary   paged_rotary: queries and keys turned by the angles of their
           positions, keys and values into their slots of the paged cache
  weights  paged_weights: the attention weight that every cached token got from
           the new ones, added to what it had
  evict    paged_evict, then paged_move of one layer: the tokens of each request
           that stay, by their weights, moved together, and the pages that get free
  verify   draft_verify: drafted tokens against the target's probabilities from
           given random numbers, and the token after the accepted ones

The plain form computes in 32 bits with elementary torch operations on padded
batches, in 64 where 32 lose what matters: the angles of far positions, and sums
of probabilities that a random number is compared with.  Lengths go by the case
alone, everything else by the seed too.
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NEG_INF = float("-inf")


def _cr():
    """This repository's package."""
    at = os.path.join(ROOT, "cu-roaring-bitmap_amd", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import curoaring
    return curoaring


def listed():
    return [
        # The new token of each of 64 requests, far into their contexts: latency.
        {"name": "rotary_decode_64", "op": "rotary", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128,
         "interleaved": False, "factor": 1.0, "far": 131072, "page": 16, "dtype": "bf16"},
        # A prefill, an odd number of tokens, half of each head turned in pairs, scaled for eight times the context.
        {"name": "rotary_prefill_30011", "op": "rotary", "tokens": 30011, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotated": 64, "interleaved": True, "factor": 8.0, "far": 1 << 20, "page": 64, "dtype": "f16"},
        # One request's token over a short context: latency.
        {"name": "weights_1x1003", "op": "weights", "requests": 1, "new": 1, "kv": 1003, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0, "past": True},
        # A decoding batch of ragged contexts up to 16384 tokens, each step added to the weights so far.
        {"name": "weights_64x16384", "op": "weights", "requests": 64, "new": 1, "kv": 16384, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0, "past": True},
        # Ragged prompts of which the last tokens, 96 dimensions wide, judge the ones that a filter lets through.
        {"name": "weights_8x100x8192_filtered", "op": "weights", "requests": 8, "new": 100, "kv": 8192, "ragged": True,
         "heads": 24, "kv_heads": 8, "dim": 96, "page": 64, "dtype": "f16", "density": 0.6, "past": False},
        # A whole prompt judged by all of its tokens: compute.
        {"name": "weights_prompt_1x16384", "op": "weights", "requests": 1, "new": 16384, "kv": 16384, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0, "past": False},
        # One request that grew a little over what it may keep: latency.
        {"name": "evict_1x1003", "op": "evict", "requests": 1, "kv": 1003, "ragged": False, "keep": 900, "sinks": 4,
         "recent": 64, "pinned": 0.0, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # A batch cut to 8192 tokens a request, some of them over it.
        {"name": "evict_64x16384", "op": "evict", "requests": 64, "kv": 16384, "ragged": True, "keep": 8192, "sinks": 4,
         "recent": 256, "pinned": 0.02, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # Long contexts cut to an eighth, pinned passages left in.
        {"name": "evict_4x131072", "op": "evict", "requests": 4, "kv": 131072, "ragged": False, "keep": 16384, "sinks": 16,
         "recent": 1024, "pinned": 0.05, "kv_heads": 4, "dim": 64, "page": 64, "dtype": "f16"},
        # One answer's four drafted tokens.
        {"name": "verify_1x4x32000", "op": "verify", "requests": 1, "drafts": 4, "ragged": False, "vocab": 32000,
         "dtype": "f32", "draft": True, "temperature": 1.0, "density": 1.0},
        # 64 answers of up to four drafts over an odd vocabulary of which a fifth may be used.
        {"name": "verify_64x4x100003", "op": "verify", "requests": 64, "drafts": 4, "ragged": True, "vocab": 100003,
         "dtype": "bf16", "draft": True, "temperature": 0.7, "density": 0.2},
        # Drafts that were looked up and have no probabilities of their own.
        {"name": "verify_128x3x64000_looked_up", "op": "verify", "requests": 128, "drafts": 3, "ragged": True,
         "vocab": 64000, "dtype": "f16", "draft": False, "temperature": 1.0, "density": 1.0},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: 1 to 128 requests, contexts of 1 to 131072 tokens, 1 to 16384 of them new, positions up to 2^20,
    vocabularies of 1000 to 100003, 0 to 8 drafts."""
    op = rng.choice(["rotary", "weights", "weights", "evict", "verify"])
    page = rng.choice([8, 16, 32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rotary":
        return {"op": op, "tokens": _log_uniform(rng, 1, 30011 * 4 // (kv_heads * group)), "heads": kv_heads * group,
                "kv_heads": kv_heads, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2]),
                "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, round(rng.uniform(1, 32), 2)]),
                "far": _log_uniform(rng, 16, 1 << 20), "page": page, "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "verify":
        requests, drafts = _log_uniform(rng, 1, 64), rng.randint(0, 8)
        vocab = _log_uniform(rng, 1000, 100003)
        requests = max(1, min(requests, 64 * 5 * 100003 // ((drafts + 1) * vocab)))
        return {"op": op, "requests": requests, "drafts": drafts, "ragged": rng.random() < 0.5, "vocab": vocab,
                "dtype": rng.choice(["bf16", "f16"] + ["f32"] * (requests <= 32)), "draft": rng.random() < 0.7,
                "temperature": rng.choice([1.0, round(rng.uniform(0.3, 1.5), 2)]),
                "density": rng.choice([1.0, round(rng.uniform(0.05, 0.9), 3)])}
    requests, kv = _log_uniform(rng, 1, 128), _log_uniform(rng, 1, 131072)
    # a cache of at most 2 GB
    while requests * kv * kv_heads * dim * 4 > 2e9:
        requests, kv = max(1, requests // 2), max(1, kv - kv // 4)
    if op == "evict":
        return {"op": op, "requests": requests, "kv": kv, "ragged": rng.random() < 0.75,
                "keep": max(1, int(kv * rng.uniform(0.05, 1.0))), "sinks": rng.randint(0, 16),
                "recent": _log_uniform(rng, 1, 1024), "pinned": rng.choice([0.0, round(rng.uniform(0.0, 0.1), 3)]),
                "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": rng.choice(["bf16", "f16", "f32"])}
    new = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 16384)
    new = min(new, kv)
    while requests * new * kv * kv_heads * group * max(1.0, dim / 128) > 16384 * 16384 * 8:
        new, requests = max(1, new - new // 3), max(1, requests - requests // 4)
    return {"op": op, "requests": requests, "new": new, "kv": kv, "ragged": rng.random() < 0.75,
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "density": rng.choice([1.0, 1.0, round(rng.uniform(0.02, 0.9), 3)]), "past": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------
def _generator(seed, part=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + part)
    return g


def _lengths(case):
    """Each request's length and new tokens (drafts and one more where it verifies), by the case's own values."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["requests"]
    if case["op"] == "verify":
        return None, [1 + (case["drafts"] if i == 0 or not case["ragged"] else rng.randint(0, case["drafts"]))
                      for i in range(n)]
    most = case.get("new", 0)
    new = [most if i == 0 or not case["ragged"] else rng.randint(1, most) if most else 0 for i in range(n)]
    return [case["kv"] if i == 0 or not case["ragged"] else rng.randint(max(1, new[i]), case["kv"])
            for i in range(n)], new


def _ceil(a, b):
    return -(-a // b)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, device="cuda", dtype=dtype)


class _Held:
    """Owns a device bitmap: freed when dropped."""

    def __init__(self, g):
        self.g = g

    def __del__(self):
        try:
            _cr().free_async(self.g)
        except Exception:
            pass


def _bitmap(mask):
    """The set bits of `mask` as the handle that a program keeps: the library's bitmap where its own calls run, and
    nothing beside the mask where the plain form does."""
    if not own:
        return None
    cr = _cr()
    n = mask.numel()
    pad = torch.zeros(_ceil(n, 32) * 32, device="cuda", dtype=torch.int64)
    pad[:n] = mask
    words = (pad.view(-1, 32) << torch.arange(32, device="cuda")).sum(1)
    words = torch.where(words > 0x7FFFFFFF, words - (1 << 32), words).to(torch.int32)
    return _Held(cr.upload_from_device_bitset(words, n))


def _random(shape, dtype, g, scale=1.0):
    x = torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g)
    return x.mul_(scale) if scale != 1.0 else x


def _tables(case, kv, g):
    """Each request's pages, scattered over the pool: (block table, pages in the pool)."""
    page = case["page"]
    held = [_ceil(n, page) for n in kv]
    pages = sum(held) + sum(held) // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    cols = max(held)
    counts = _ints(held, torch.int64)
    first = torch.cumsum(counts, 0) - counts
    col = torch.arange(cols, device="cuda")
    at = (first[:, None] + col).clamp(max=pages - 1)
    return torch.where(col < counts[:, None], order[at], -1).to(torch.int32), pages


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = {"case": case}
    page = case.get("page")
    if op == "rotary":
        dt, n, rot = DTYPES[case["dtype"]], case["tokens"], case["rotated"]
        pages = _ceil(n, page) + _ceil(n, page) // 4 + 1
        order = torch.randperm(pages, generator=g, device="cuda")[:_ceil(n, page)]
        s["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n].contiguous()
        s["q"] = _random((n, case["heads"], case["dim"]), dt, g)
        s["k"] = _random((n, case["kv_heads"], case["dim"]), dt, g)
        s["v"] = _random((n, case["kv_heads"], case["dim"]), dt, g)
        s["q_out"] = torch.empty_like(s["q"])
        s["k_cache"] = torch.zeros(pages, page, case["kv_heads"], case["dim"], device="cuda", dtype=dt)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        # runs of neighbouring tokens, each somewhere in its context
        run = max(1, n // 64)
        base = torch.randint(0, case["far"], (_ceil(n, run),), generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        s["positions"] = (base[at // run] + at % run).to(torch.int32)
        # slow pairs are slowed further for long contexts, fast ones left
        i = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64)
        slow = (i / max(1, rot - 2)).clamp(0, 1)
        s["freqs"] = 10000.0 ** (-i / rot) * (1 - slow + slow / case["factor"])
        s["magnitude"] = 1.0 + 0.1 * math.log(case["factor"])
    elif op == "weights":
        kv, new = _lengths(case)
        dt, total = DTYPES[case["dtype"]], sum(new)
        s["table"], pages = _tables(case, kv, g)
        s["k_cache"] = _random((pages, page, case["kv_heads"], case["dim"]), dt, g)
        # scores of a few units' spread, as trained attention has
        s["q"] = _random((total, case["heads"], case["dim"]), dt, g, 2.5)
        s["starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["kv_len"] = _ints(kv)
        s["max_new"], s["max_kv"] = max(new), max(kv)
        s["visible"] = s["filter"] = None
        if case["density"] < 1:
            # pages of documents that pass, and a few single slots of the others
            by_page = torch.rand(pages, device="cuda", generator=g) < case["density"]
            by_slot = torch.rand(pages * page, device="cuda", generator=g) < 0.02
            s["visible"] = by_page.repeat_interleave(page) ^ by_slot
            s["filter"] = _bitmap(s["visible"])
        shape = (len(new), s["table"].shape[1] * page)
        s["past"] = 4 * torch.rand(shape, device="cuda", generator=g) if case["past"] else None
        s["out"] = torch.zeros(shape, device="cuda")
        s["lse"] = _log_sums(s)
    elif op == "evict":
        kv, _ = _lengths(case)
        dt, n = DTYPES[case["dtype"]], case["requests"]
        s["table"], pages = _tables(case, kv, g)
        room = s["table"].shape[1] * page
        s["k_cache"] = _random((pages, page, case["kv_heads"], case["dim"]), dt, g)
        s["v_cache"] = _random((pages, page, case["kv_heads"], case["dim"]), dt, g)
        s["kv_len"] = _ints(kv)
        # a few tokens are looked at much, some never
        w = torch.randn(n, room, device="cuda", generator=g).mul_(2).exp_()
        s["weights"] = torch.where(torch.rand(n, room, device="cuda", generator=g) < 0.05, 0.0, w)
        # what is left of twice as many tokens, out of order, and the ones that came since
        share = torch.rand(n, device="cuda", generator=g)
        s["kept"] = (share * s["kv_len"]).to(torch.int32)
        turn = torch.randint(0, 1 << 30, (n, 1), device="cuda", generator=g)
        odd = torch.randint(0, 2, (n, room), device="cuda", generator=g)
        i = torch.arange(room, device="cuda")
        s["positions"] = (2 * ((i + turn) % s["kept"][:, None].clamp(min=1)) + odd).to(torch.int32)
        s["seen"] = s["kept"] + s["kv_len"]
        s["keep"] = torch.full((n,), case["keep"], device="cuda", dtype=torch.int32)
        s["pinned"] = s["pins"] = None
        if case["pinned"]:
            s["pinned"] = torch.rand(pages * page, device="cuda", generator=g) < case["pinned"]
            s["pins"] = _bitmap(s["pinned"])
        s["weights_out"] = torch.zeros(n, room, device="cuda")
        s["positions_out"] = torch.zeros(n, room, device="cuda", dtype=torch.int32)
        s["len"] = torch.zeros(n, device="cuda", dtype=torch.int32)
        s["moves"] = torch.full((n, _ceil(room, 2), 2), -1, device="cuda", dtype=torch.int32)
        s["n_moves"] = torch.zeros(n, device="cuda", dtype=torch.int32)
        s["freed"] = torch.full((sum(_ceil(x, page) for x in kv),), -1, device="cuda", dtype=torch.int32)
        s["counts"] = torch.zeros(2, device="cuda", dtype=torch.int32)
    else:
        _, rows = _lengths(case)
        n, total, vocab, dt = len(rows), sum(rows), case["vocab"], DTYPES[case["dtype"]]
        s["starts"] = _ints([sum(rows[:i]) for i in range(n + 1)])
        x = _random((total, vocab), torch.float32, g, 2.5)
        s["scores"] = x.to(dt)
        # the drafting model thinks much the same, and draws its tokens from what it thinks
        x = x.add_(_random((total, vocab), torch.float32, g, 0.7))
        s["mask"] = s["allowed"] = None
        if case["density"] < 1:
            s["mask"] = torch.rand(vocab, device="cuda", generator=g) < case["density"]
            s["allowed"] = _bitmap(s["mask"])
        s["draft"] = x.to(dt) if case["draft"] else None
        x = x.div_(case["temperature"])
        x = x - torch.log(-torch.log(torch.rand(total, vocab, device="cuda", generator=g).clamp_(1e-20, 1 - 1e-7)))
        if s["mask"] is not None:
            x = torch.where(s["mask"], x, NEG_INF)
        # the step's tokens: the one that draft j was drawn for comes after token j
        first = torch.randint(0, vocab, (1,), device="cuda", generator=g)
        s["tokens"] = torch.cat([first, x.argmax(1)[:-1]]).to(torch.int32)
        s["uniform"] = torch.rand(total, device="cuda", generator=g)
        s["accepted"] = torch.zeros(n, device="cuda", dtype=torch.int32)
        s["out"] = torch.zeros(n, max(rows), device="cuda", dtype=torch.int32)
    return s


def _padded(s):
    """Queries, keys and masks of the requests side by side: q [R * key heads, heads of a group * new, dim], k
    [R * key heads, dim, n], which keys each new token sees [R, new, n], and each new token's place in q."""
    case = s["case"]
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    group, requests, total = case["heads"] // kv_heads, case["requests"], s["q"].shape[0]
    kv_len, starts = s["kv_len"].long(), s["starts"].long()
    new, m, n = starts[1:] - starts[:-1], s["max_new"], s["max_kv"]
    pos, tok = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    slot = s["table"].long()[:, pos // page].clamp(min=0) * page + pos % page
    last = kv_len[:, None] - new[:, None] + tok  # the position of each new token
    sees = (pos < kv_len[:, None])[:, None] & (pos <= last[:, :, None]) & (tok < new[:, None])[:, :, None]
    if s["visible"] is not None:
        sees &= s["visible"][slot][:, None]
    k = s["k_cache"].view(-1, kv_heads, dim)[slot].permute(0, 2, 3, 1).float().reshape(-1, dim, n)
    place = (starts[:-1, None] + tok).clamp(max=total - 1)
    q = s["q"][place].float().view(requests, m, kv_heads, group, dim)
    return q.permute(0, 2, 3, 1, 4).reshape(requests * kv_heads, group * m, dim), k, sees, place


def _log_sums(s):
    """What the attention of these queries leaves beside its output: log(sum(exp(scale * q k))) [tokens, heads]."""
    case = s["case"]
    kv_heads, heads, requests = case["kv_heads"], case["heads"], case["requests"]
    q, k, sees, _ = _padded(s)
    group, m, n = heads // kv_heads, s["max_new"], s["max_kv"]
    q = q.view(requests, kv_heads, group * m, -1)
    k = k.view(requests, kv_heads, -1, n)
    out = torch.empty(requests, heads, m, device="cuda")
    for h in range(kv_heads):
        x = torch.bmm(q[:, h].contiguous(), k[:, h].contiguous()).mul_(case["dim"] ** -0.5)
        x = x.view(requests, group, m, n).masked_fill_(~sees[:, None], NEG_INF)
        out[:, h * group:(h + 1) * group] = torch.logsumexp(x, 3)
    starts = s["starts"].long()
    r = torch.repeat_interleave(torch.arange(requests, device="cuda"), starts[1:] - starts[:-1])
    return out[r, :, torch.arange(s["q"].shape[0], device="cuda") - starts[r]].contiguous()


# ---- one pass ------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"rotary": _rotary, "weights": _weights, "evict": _evict, "verify": _verify}[op](state)
    cr, s = _cr(), state
    case = s["case"]
    if op == "rotary":
        cr.paged_rotary(s["k"], s["v"], s["positions"], s["freqs"], s["slots"], s["k_cache"], s["v_cache"], d_q=s["q"],
                        d_q_out=s["q_out"], interleaved=case["interleaved"], magnitude=s["magnitude"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "weights":
        cr.paged_weights(s["q"], s["k_cache"], s["table"], s["starts"], s["kv_len"], s["lse"], s["out"], d_past=s["past"],
                         decay=0.9, visible=s["filter"].g if s["filter"] else None, max_new=s["max_new"],
                         max_kv=s["max_kv"])
        return s["out"]
    if op == "evict":
        cr.paged_evict(s["weights"], s["kv_len"], s["keep"], s["table"], case["page"], s["weights_out"], s["len"],
                       s["moves"], s["n_moves"], s["freed"], s["counts"], d_positions=s["positions"], d_kept=s["kept"],
                       d_seen=s["seen"], d_positions_out=s["positions_out"], sinks=case["sinks"], recent=case["recent"],
                       pinned=s["pins"].g if s["pins"] else None, n_pages=s["k_cache"].shape[0])
        cr.paged_move(s["moves"], s["n_moves"], s["k_cache"], s["v_cache"])
        return {x: s[x] for x in ("weights_out", "positions_out", "len", "moves", "n_moves", "freed", "counts", "k_cache",
                                  "v_cache")}
    cr.draft_verify(s["scores"], s["tokens"], s["starts"], s["uniform"], s["accepted"], s["out"], d_draft=s["draft"],
                    temperature=case["temperature"], allowed=s["allowed"].g if s["allowed"] else None)
    return {"accepted": s["accepted"], "out": s["out"]}


def _rotary(s):
    case = s["case"]
    rot, dim = case["rotated"], case["dim"]
    angle = s["positions"].double()[:, None] * s["freqs"]
    c, d = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2),
                                                                                      slice(rot // 2, rot))

    def turned(x):
        x, out = x.float(), x.clone()
        out[..., first] = (x[..., first] * c - x[..., second] * d).to(out.dtype)
        out[..., second] = (x[..., second] * c + x[..., first] * d).to(out.dtype)
        return out

    s["k_cache"].view(-1, case["kv_heads"], dim)[s["slots"]] = turned(s["k"])
    s["v_cache"].view(-1, case["kv_heads"], dim)[s["slots"]] = s["v"]
    return {"q": turned(s["q"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _weights(s):
    case = s["case"]
    requests, heads, kv_heads, m, n = case["requests"], case["heads"], case["kv_heads"], s["max_new"], s["max_kv"]
    q, k, sees, place = _padded(s)
    lse = s["lse"][place].permute(0, 2, 1)[..., None]  # [R, heads, new, 1]
    x = torch.bmm(q, k).mul_(case["dim"] ** -0.5).view(requests, heads, m, n)
    x = x.sub_(torch.where(lse == NEG_INF, 0.0, lse)).masked_fill_(~sees[:, None], NEG_INF).exp_()
    got = x.sum((1, 2))
    pos, kv_len, new = torch.arange(n, device="cuda"), s["kv_len"].long(), s["starts"][1:] - s["starts"][:-1]
    if s["past"] is not None:
        got = got + torch.where(pos < (kv_len - new)[:, None], s["past"][:, :n] * 0.9, 0.0)
    s["out"][:, :n] = torch.where(pos < kv_len[:, None], got, s["out"][:, :n])
    return s["out"]


def _evict(s):
    case = s["case"]
    page, table = case["page"], s["table"].long()
    requests, room = s["weights"].shape
    i, n = torch.arange(room, device="cuda"), s["kv_len"].long()[:, None]
    seen, there = s["seen"].long()[:, None], i < s["kv_len"][:, None]
    position = torch.where(i < s["kept"][:, None], s["positions"].long(), seen - n + i)
    slot = table[:, i // page] * page + i % page
    safe = (position < case["sinks"]) | (position >= seen - case["recent"])
    if s["pinned"] is not None:
        safe |= s["pinned"][slot.clamp(min=0)]
    safe &= there
    keep = torch.maximum(torch.minimum(n, s["keep"].long()[:, None].clamp(min=0)), safe.sum(1, keepdim=True))
    # the order of (safe, weight, lowest place first) as whole numbers; weights are not negative here
    key = torch.where(safe, 1 << 32, s["weights"].view(torch.int32).long())
    key = torch.where(there, key, -1)
    order = torch.sort(key, dim=1, descending=True, stable=True)[1]
    stays = torch.zeros_like(there).scatter_(1, order, i < keep)
    hole, moved = (i < keep) & ~stays, (i >= keep) & stays
    # hole j of a request takes the j-th of its tokens that stay and lie behind
    r, to = torch.nonzero(hole, as_tuple=True)
    rank = (torch.cumsum(hole, 1) - 1)[r, to]
    source = torch.nonzero(moved, as_tuple=True)[1]
    moves = torch.full_like(s["moves"], -1)
    moves[r, rank, 0], moves[r, rank, 1] = slot[r, source].to(torch.int32), slot[r, to].to(torch.int32)
    weights, position = s["weights"].clone(), position.to(torch.int32)
    weights[r, to], position[r, to] = s["weights"][r, source], position[r, source]
    kept = i < keep
    weights, position = (torch.where(kept, x, y) for x, y in ((weights, s["weights_out"]),
                                                              (position, s["positions_out"])))
    col = torch.arange(table.shape[1], device="cuda")
    free = table[(col >= (keep + page - 1) // page) & (col < (n + page - 1) // page)]
    freed = torch.full_like(s["freed"], -1)
    freed[:free.numel()] = free.to(torch.int32)
    for t in (s["k_cache"], s["v_cache"]):
        t = t.view(-1, case["kv_heads"], case["dim"])
        t[slot[r, to]] = t[slot[r, source]]
    n_moves = hole.sum(1).to(torch.int32)
    counts = torch.tensor([free.numel(), r.numel()], device="cuda", dtype=torch.int32)
    return {"weights_out": weights, "positions_out": position, "len": keep[:, 0].to(torch.int32), "moves": moves,
            "n_moves": n_moves, "freed": freed, "counts": counts, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _probabilities(x, temperature, mask):
    x = x.double() / temperature
    x = torch.where(torch.isnan(x) if mask is None else torch.isnan(x) | ~mask, NEG_INF, x)
    top = x.amax(1, keepdim=True)
    x = x.sub_(torch.where(top == NEG_INF, 0.0, top)).exp_()
    mass = x.sum(1, keepdim=True)
    return x.div_(torch.where(mass > 0, mass, 1.0))


def _verify(s):
    case, starts, token = s["case"], s["starts"].long(), s["tokens"].long()
    total, vocab = s["scores"].shape
    most = s["out"].shape[1]
    p = _probabilities(s["scores"], case["temperature"], s["mask"])
    follows = torch.roll(token, -1)  # what was drafted after each token
    at = torch.arange(vocab, device="cuda")
    if s["draft"] is not None:
        q = _probabilities(s["draft"], case["temperature"], s["mask"])
    else:
        q = (at == follows[:, None]).double()
    u = s["uniform"].double()
    pick = follows[:, None]
    good = u * q.gather(1, pick)[:, 0] < p.gather(1, pick)[:, 0]
    j = torch.arange(most, device="cuda")
    drafts = (starts[1:] - starts[:-1] - 1)[:, None]
    row = (starts[:-1, None] + j).clamp(max=total - 1)
    accepted = torch.cumprod((good[row] & (j < drafts)).long(), 1).sum(1, keepdim=True)
    stop = (starts[:-1, None] + accepted)[:, 0]
    p, q = p[stop], q[stop]
    rest = torch.where(accepted < drafts, (p - q).clamp(min=0), p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    upto = torch.cumsum(rest, 1)
    may = rest > 0
    over = may & (upto > u[starts[1:] - 1][:, None] * upto[:, -1:])
    first = torch.where(over, at, vocab).amin(1)
    last = torch.where(may, at, -1).amax(1)
    token = torch.where(first < vocab, first, last)[:, None]
    out = torch.where(j < accepted, follows[row], torch.where(j == accepted, token, -1))
    return {"accepted": accepted[:, 0].to(torch.int32), "out": out.to(torch.int32)}


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "rotary":
        n, heads, kv_heads, dim, rot = (case[x] for x in ("tokens", "heads", "kv_heads", "dim", "rotated"))
        return {"bytes": n * (2 * size * dim * (heads + 2 * kv_heads) + 12) + 4 * rot,
                "flops": 3 * n * rot * (heads + kv_heads)}
    if op == "verify":
        rows = sum(_lengths(case)[1])
        read = rows + (rows - case["requests"] if case["draft"] else 0)
        bits = case["vocab"] / 8 if case["density"] < 1 else 0
        return {"bytes": read * case["vocab"] * size + bits + 12 * rows, "flops": 3 * read * case["vocab"]}
    kv, new = _lengths(case)
    held = sum(_ceil(n, case["page"]) for n in kv)
    if op == "weights":
        share = case["density"] * 0.96 + 0.02 if case["density"] < 1 else 1.0  # what passes, single slots included
        keys = sum(kv) * share
        pairs = sum(m * (n - m) + m * (m + 1) / 2 for n, m in zip(kv, new)) * share
        marks = held * case["page"] / 8 if case["density"] < 1 else 0
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] + sum(new) * case["heads"] * (2 * case["dim"] + 4) +
                4 * held + marks + sum(kv) * (8 if case["past"] else 4), "flops": 2 * pairs * case["heads"] * case["dim"]}
    left = [min(n, case["keep"]) for n in kv]
    # of the tokens that stay, as many lie behind as are let go of before: what stays is anywhere
    moves = sum(m * (n - m) / n for n, m in zip(kv, left))
    marks = held * case["page"] / 8 if case["pinned"] else 0
    return {"bytes": sum(kv) * 6 + marks + 4 * held + sum(left) * 8 + moves * (8 + 4 * size * case["kv_heads"] * case["dim"]),
            "flops": 2 * sum(kv)}


def exact(case, seed):
    """The computed numbers in 64 bits; whole numbers and moved rows have no such value."""
    if case["op"] in ("evict", "verify"):
        return None
    s = prepare(case, seed)
    page, kv_heads = case["page"], case["kv_heads"]
    if case["op"] == "rotary":
        rot = case["rotated"]
        turns = torch.outer(s["positions"].double(), s["freqs"])
        spin = torch.polar(torch.full_like(turns, s["magnitude"]), turns)[:, None]

        def turned(x):
            x = x.double()
            y = x[..., :rot]
            y = y.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else y.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * spin)
            y = y if case["interleaved"] else y.transpose(-1, -2)
            return torch.cat([y.flatten(-2), x[..., rot:]], -1)

        k, v = s["k_cache"].double(), s["v_cache"].double()
        at = s["slots"] // page, s["slots"] % page
        k[at], v[at] = turned(s["k"]), s["v"].double()
        return {"q": turned(s["q"]), "k_cache": k, "v_cache": v}
    group = case["heads"] // kv_heads
    kc = s["k_cache"].view(-1, kv_heads, case["dim"])
    out = s["out"].double()
    kv, new = _lengths(case)
    at = 0
    for r, (c, n) in enumerate(zip(kv, new)):
        here = torch.arange(c, device="cuda")
        slot = s["table"][r, here // page].long() * page + here % page
        mine = torch.zeros(c, device="cuda", dtype=torch.float64)
        for h in range(kv_heads):
            k = kc[slot, h].double()
            for i in range(0, n, 2048):
                j = min(n, i + 2048)
                q = s["q"][at + i:at + j, h * group:(h + 1) * group].double()
                p = torch.einsum("tgd,kd->gtk", q, k) / math.sqrt(case["dim"])
                z = s["lse"][at + i:at + j, h * group:(h + 1) * group].t().double()[:, :, None]
                p = torch.exp(p - torch.where(z == NEG_INF, 0.0, z))
                seen = here <= c - n + torch.arange(i, j, device="cuda")[:, None]
                if s["visible"] is not None:
                    seen = seen & s["visible"][slot]
                mine += torch.where(seen, p, 0.0).sum((0, 1))
        if s["past"] is not None:
            mine[:c - n] += 0.9 * s["past"][r, :c - n].double()
        out[r, :c] = mine
        at += n
    return out
