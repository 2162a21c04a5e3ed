"""The library's operators for serving language models, as measurable cases.

A server keeps sets of ids next to its paged key/value cache: free pages, slots
that a request may look at, tokens that an answer may use.  A case is a dict of
plain values; `op` says which operator one pass runs:

  plan       paged_plan: block tables and slot maps from request lengths, the
             pages taken from a bitmap of free ones
  append     paged_append: new keys and values into their slots
  attention  paged_attention: new tokens (one or a chunk a request) over the
             paged cache; with `density` < 1 a bitmap says which slots are
             visible, and paged_select lists them first
  beam       beam_select over beams and vocabulary, then beam_reorder of the
             beams' states

The plain form computes in 32 bits with elementary torch operations on padded
batches.  Lengths go by the case alone, everything else by the seed too.
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
        # A decoding step of a small server: a token each for 64 requests, four of which need a page.
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "cached": 2000, "new": 1, "page": 16, "pages": 8192},
        # A large prefill: 1024 ragged prompts, about four million tokens, from a pool of a million pages.
        {"name": "plan_prefill_1024", "op": "plan", "requests": 1024, "cached": 4096, "new": 8192, "page": 16,
         "pages": 1 << 20},
        # The new token of each of 64 requests into the cache.
        {"name": "append_decode_64", "op": "append", "tokens": 64, "heads": 8, "dim": 128, "page": 16, "dtype": "bf16"},
        # A prefill's keys and values, an odd number of tokens.
        {"name": "append_prefill_30011", "op": "append", "tokens": 30011, "heads": 8, "dim": 128, "page": 64,
         "dtype": "f16"},
        # One request's next token over a short context: latency.
        {"name": "decode_1x1003", "op": "attention", "requests": 1, "new": 1, "kv": 1003, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0},
        # A decoding batch of ragged contexts up to 16384 tokens.
        {"name": "decode_64x16384", "op": "attention", "requests": 64, "new": 1, "kv": 16384, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0},
        # Every head with its own keys, 64 dimensions, four tokens a request to be checked at once.
        {"name": "verify_48x2048_mha", "op": "attention", "requests": 48, "new": 4, "kv": 2048, "ragged": True,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 32, "dtype": "f16", "density": 1.0},
        # Long contexts of which a filter lets an eighth through: each step looks at the passing documents only.
        {"name": "decode_4x131072_filtered", "op": "attention", "requests": 4, "new": 1, "kv": 131072, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "f16", "density": 0.125},
        # Ragged chunks over a filtered cache, 96 dimensions.
        {"name": "chunk_8x1000_filtered", "op": "attention", "requests": 8, "new": 1000, "kv": 8192, "ragged": True,
         "heads": 24, "kv_heads": 8, "dim": 96, "page": 64, "dtype": "bf16", "density": 0.6},
        # A whole prompt of 16384 tokens: compute.
        {"name": "prefill_1x16384", "op": "attention", "requests": 1, "new": 16384, "kv": 16384, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "density": 1.0},
        # One answer's four beams over log-probabilities, eight candidates kept as a search with finished beams does.
        {"name": "beam_1x4x32000", "op": "beam", "batch": 1, "beams": 4, "vocab": 32000, "k": 8, "dtype": "f32",
         "density": 1.0, "states": 4096},
        # 64 answers of eight beams over an odd vocabulary of raw scores, a fifth of the tokens allowed.
        {"name": "beam_64x8x100003", "op": "beam", "batch": 64, "beams": 8, "vocab": 100003, "k": 8, "dtype": "bf16",
         "density": 0.2, "states": 32768},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: 1 to 1024 requests, contexts of 1 to 131072 tokens, chunks of 1 to 16384, vocabularies of 1000 to
    130000."""
    op = rng.choice(["plan", "append", "attention", "attention", "attention", "beam"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "plan":
        requests, new = _log_uniform(rng, 1, 1024), _log_uniform(rng, 1, 8192)
        cached = _log_uniform(rng, 1, 8192)
        return {"op": op, "requests": requests, "cached": cached, "new": new, "page": page,
                "pages": 2 * requests * (math.ceil((cached + new) / page) + 1) + rng.randint(0, 999)}
    if op == "append":
        return {"op": op, "tokens": _log_uniform(rng, 1, 30011), "heads": rng.choice([1, 2, 4, 5, 8]),
                "dim": rng.choice([64, 80, 96, 128]), "page": page, "dtype": rng.choice(["bf16", "f16"])}
    if op == "beam":
        batch, beams = _log_uniform(rng, 1, 64), rng.randint(1, 8)
        dtypes = ["bf16", "f16", "f32"] if batch <= 32 else ["bf16", "f16"]
        return {"op": op, "batch": batch, "beams": beams, "vocab": _log_uniform(rng, 1000, 100003),
                "k": rng.choice([beams, 2 * beams]), "dtype": rng.choice(dtypes),
                "density": rng.choice([1.0, round(rng.uniform(0.05, 0.9), 3)]),
                "states": 8 * _log_uniform(rng, 16, 2048)}
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    requests = _log_uniform(rng, 1, 128)
    new = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 16384)
    kv = max(new, _log_uniform(rng, 1, 131072))
    # at most a quarter of the largest listed case's scores, and a cache of at most 4 GB
    while requests * kv * kv_heads * dim * 4 > 4e9:
        requests, kv = max(1, requests // 2), max(1, kv - kv // 4)
    new = min(new, kv)
    while requests * new * kv * kv_heads * group * max(1.0, dim / 128) > 16384 * 16384 * 8:
        new, requests = max(1, new - new // 3), max(1, requests - requests // 4)
    return {"op": op, "requests": requests, "new": new, "kv": kv, "ragged": rng.random() < 0.75,
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": rng.choice(["bf16", "f16"]), "density": rng.choice([1.0, 1.0, round(rng.uniform(0.02, 0.9), 3)])}


# ---- inputs ------------------------------------------------------------------
def _generator(seed, part=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 64 + part)
    return g


def _lengths(case):
    """(cached, new) of each request: by the case's own values, the longest first."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, most = case["requests"], case["new"]
    if case["op"] == "plan":
        return [rng.randint(0, case["cached"]) for _ in range(n)], [rng.randint(1, most) for _ in range(n)]
    new = [most if i == 0 or not case["ragged"] else rng.randint(1, most) for i in range(n)]
    kv = [case["kv"] if i == 0 or not case["ragged"] else rng.randint(new[i], case["kv"]) for i in range(n)]
    return [a - b for a, b in zip(kv, new)], new


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


def _tables(case, cached, new, g):
    """Each request's pages, scattered over the pool: (block table, pages in the pool)."""
    page = case["page"]
    held = [_ceil(c + n, page) for c, n in zip(cached, new)]
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
    if op == "plan":
        cached, new = _lengths(case)
        page, pages = case["page"], case["pages"]
        held, most = [_ceil(c, page) for c in cached], [_ceil(c + n, page) for c, n in zip(cached, new)]
        cols, total, taken = max(most), sum(new), sum(most) - sum(held)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        counts = _ints(held, torch.int64)
        col, first = torch.arange(cols, device="cuda"), torch.cumsum(counts, 0) - counts
        used = sum(held)
        s["table"] = torch.where(col < counts[:, None], order[(first[:, None] + col).clamp(max=pages - 1)],
                                 -1).to(torch.int32)
        # pages of other requests: of those left, at most as many as leave a tenth more than is needed
        spare = pages - used - taken
        busy = used + max(0, min(spare, int(0.6 * spare)))
        s["free_mask"] = torch.ones(pages, device="cuda", dtype=torch.bool)
        s["free_mask"][order[:busy].long()] = False
        s["free"] = _bitmap(s["free_mask"])
        s["cached"], s["new"] = _ints(cached), _ints(new)
        s["slots"] = torch.full((total,), -1, device="cuda", dtype=torch.int64)
        s["starts"] = torch.zeros(len(new) + 1, device="cuda", dtype=torch.int32)
        s["kv_len"] = torch.zeros(len(new), device="cuda", dtype=torch.int32)
        s["taken"] = torch.full((max(1, taken),), -1, device="cuda", dtype=torch.int32)
        s["counts"] = torch.zeros(3, device="cuda", dtype=torch.int32)
    elif op == "append":
        dt, n, page = DTYPES[case["dtype"]], case["tokens"], case["page"]
        pages = _ceil(n, page) + _ceil(n, page) // 4 + 1
        # whole pages in scattered order, the last one in part
        order = torch.randperm(pages, generator=g, device="cuda")[:_ceil(n, page)]
        s["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n].contiguous()
        s["k"] = _random((n, case["heads"], case["dim"]), dt, g)
        s["v"] = _random((n, case["heads"], case["dim"]), dt, g)
        s["k_cache"] = torch.zeros(pages, page, case["heads"], case["dim"], device="cuda", dtype=dt)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
    elif op == "attention":
        cached, new = _lengths(case)
        dt, page, total = DTYPES[case["dtype"]], case["page"], sum(new)
        s["table"], pages = _tables(case, cached, new, g)
        s["k_cache"] = _random((pages, page, case["kv_heads"], case["dim"]), dt, g)
        s["v_cache"] = _random((pages, page, case["kv_heads"], case["dim"]), dt, g)
        # scores of a few units' spread, as trained attention has
        s["q"] = _random((total, case["heads"], case["dim"]), dt, g, 2.5)
        s["starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["kv_len"] = _ints([c + n for c, n in zip(cached, new)])
        s["max_new"], s["max_kv"] = max(new), max(c + n for c, n in zip(cached, new))
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(total, case["heads"], device="cuda")
        if case["density"] < 1:
            # pages of documents that pass, and a few single slots of the others
            by_page = torch.rand(pages, device="cuda", generator=g) < case["density"]
            by_slot = torch.rand(pages * page, device="cuda", generator=g) < 0.02
            s["visible"] = by_page.repeat_interleave(page) ^ by_slot
            s["filter"] = _bitmap(s["visible"])
            s["sel"] = torch.zeros(len(new), s["table"].shape[1] * page, device="cuda", dtype=torch.int32)
            s["sel_len"] = torch.zeros(len(new), device="cuda", dtype=torch.int32)
            s["limits"] = torch.zeros(total, device="cuda", dtype=torch.int32)
    else:
        b, w, v, k = case["batch"], case["beams"], case["vocab"], case["k"]
        dt = DTYPES[case["dtype"]]
        x = _random((b, w, v), torch.float32, g, 2.5)
        s["lse"] = None
        if dt == torch.float32:
            x = x - torch.logsumexp(x, 2, keepdim=True)
        x = x.to(dt)
        if dt != torch.float32:  # raw scores, with the normaliser that the program's output layer left
            s["lse"] = torch.logsumexp(x.float(), 2).contiguous()
        s["x"] = x
        s["cum"] = -8 * torch.rand(b, w, device="cuda", generator=g)
        s["mask"] = s["allowed"] = None
        if case["density"] < 1:
            s["mask"] = torch.rand(v, device="cuda", generator=g) < case["density"]
            s["allowed"] = _bitmap(s["mask"])
        s["scores"] = torch.empty(b, k, device="cuda")
        s["tokens"] = torch.empty(b, k, device="cuda", dtype=torch.int32)
        s["parents"] = torch.empty(b, k, device="cuda", dtype=torch.int32)
        s["states"] = _random((b, w, case["states"] // 8, 8), torch.bfloat16, g)
        s["next"] = torch.zeros(b, k, case["states"] // 8, 8, device="cuda", dtype=torch.bfloat16)
        s["len"] = torch.randint(1, case["states"] // 8 + 1, (b, w), device="cuda", generator=g).to(torch.int32)
    return s


# ---- one pass ------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan, "append": _append, "attention": _attention, "beam": _beam}[op](state)
    cr, s = _cr(), state
    case = s["case"]
    if op == "plan":
        cr.paged_plan(s["free"].g, case["pages"], case["page"], s["cached"], s["new"], s["table"], s["slots"],
                      s["starts"], s["kv_len"], s["taken"], s["counts"])
        return {x: s[x] for x in ("table", "slots", "starts", "kv_len", "taken", "counts")}
    if op == "append":
        cr.paged_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "attention":
        got, selection = {"out": s["out"], "lse": s["lse"]}, None
        if "visible" in s:
            selection = (s["sel"], s["sel_len"], s["limits"])
            cr.paged_select(s["filter"].g, s["table"], s["starts"], s["kv_len"], case["page"], *selection)
            got |= {"sel": s["sel"], "sel_len": s["sel_len"], "limits": s["limits"]}
        cr.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["kv_len"], s["out"],
                           scale=case["dim"] ** -0.5, d_lse=s["lse"], selection=selection, max_new=s["max_new"],
                           max_kv=s["max_kv"])
        return got
    cr.beam_select(s["x"], s["cum"], s["scores"], s["tokens"], s["parents"], d_lse=s["lse"],
                   allowed=s["allowed"].g if s["allowed"] else None)
    cr.beam_reorder(s["states"], s["parents"], s["next"], d_len=s["len"])
    return {x: s[x] for x in ("scores", "tokens", "parents", "next")}


def _plan(s):
    page, cached, new, table = s["case"]["page"], s["cached"].long(), s["new"].long(), s["table"]
    requests, cols = table.shape
    pages = s["free_mask"].numel()
    held, most = (cached + page - 1) // page, (cached + new + page - 1) // page
    need = most - held
    upto = torch.cumsum(need, 0)
    # the free pages' ids, ascending, then the others'
    ids = torch.sort(torch.where(s["free_mask"], 0, pages) + torch.arange(pages, device="cuda"))[0] % pages
    granted = (need == 0) | (upto <= s["free_mask"].sum())
    col = torch.arange(cols, device="cuda")
    fresh = (col >= held[:, None]) & (col < most[:, None]) & granted[:, None]
    rank = (upto - need)[:, None] + col - held[:, None]
    out = torch.where(fresh, ids[rank.clamp(0, pages - 1)], table.long())
    starts = torch.cumsum(torch.cat([torch.zeros_like(new[:1]), new]), 0)
    total = s["slots"].numel()
    r = torch.repeat_interleave(torch.arange(requests, device="cuda"), new, output_size=total)
    at = cached[r] + torch.arange(total, device="cuda") - starts[r]
    slots = torch.where(granted[r], out[r, (at // page).clamp(max=cols - 1)] * page + at % page, -1)
    taken = torch.where(granted, need, 0).sum()
    rank = torch.arange(s["taken"].numel(), device="cuda")
    return {"table": out.to(torch.int32), "slots": slots, "starts": starts.to(torch.int32),
            "kv_len": torch.where(granted, cached + new, 0).to(torch.int32),
            "taken": torch.where(rank < taken, ids[rank.clamp(max=pages - 1)], -1).to(torch.int32),
            "counts": torch.stack([starts[-1], taken, need.sum() - taken]).to(torch.int32)}


def _append(s):
    pages, page, heads, dim = s["k_cache"].shape
    s["k_cache"].view(-1, heads, dim)[s["slots"]] = s["k"]
    s["v_cache"].view(-1, heads, dim)[s["slots"]] = s["v"]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    case = s["case"]
    page, heads, kv_heads, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    group, requests, total = heads // kv_heads, case["requests"], s["q"].shape[0]
    kv_len, starts = s["kv_len"].long(), s["starts"].long()
    new, m, n = starts[1:] - starts[:-1], s["max_new"], s["max_kv"]
    pos, tok = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    slot = s["table"].long()[:, pos // page].clamp(min=0) * page + pos % page
    last = kv_len[:, None] - new[:, None] + tok  # the position of each new token
    there = pos < kv_len[:, None]
    got = {}
    if "visible" in s:
        there = there & s["visible"][slot]
        upto = torch.cumsum(there, 1)
        room = s["sel"].shape[1]
        sel = torch.zeros(requests, room + 1, device="cuda", dtype=torch.int32)
        sel.scatter_(1, torch.where(there, upto - 1, room), slot.to(torch.int32))
        of = torch.repeat_interleave(torch.arange(requests, device="cuda"), new, output_size=total)
        at = last[of, torch.arange(total, device="cuda") - starts[of]]
        got = {"sel": sel[:, :room].contiguous(), "sel_len": there.sum(1).to(torch.int32),
               "limits": upto[of, at].to(torch.int32)}
    k = s["k_cache"].view(-1, kv_heads, dim)[slot].permute(0, 2, 3, 1).float().reshape(-1, dim, n)
    v = s["v_cache"].view(-1, kv_heads, dim)[slot].permute(0, 2, 1, 3).float().reshape(-1, n, dim)
    q = s["q"][(starts[:-1, None] + tok).clamp(max=total - 1)].float().view(requests, m, kv_heads, group, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(requests * kv_heads, group * m, dim)
    x = torch.bmm(q, k).mul_(dim ** -0.5).view(requests, kv_heads * group, m, n)
    x.masked_fill_(~(there[:, None] & (pos <= last[:, :, None]))[:, None], NEG_INF)
    top = x.amax(3, keepdim=True)
    top = torch.where(top == NEG_INF, 0.0, top)
    x = x.sub_(top).exp_()
    mass = x.sum(3, keepdim=True)
    o = torch.bmm(x.view(requests * kv_heads, group * m, n), v).view(requests, heads, m, dim)
    o = torch.where(mass > 0, o / mass, 0.0)
    lse = (top + torch.log(mass))[..., 0]
    r = torch.repeat_interleave(torch.arange(requests, device="cuda"), new, output_size=total)
    i = torch.arange(total, device="cuda") - starts[r]
    return {"out": o[r, :, i].to(s["q"].dtype), "lse": lse[r, :, i].contiguous(), **got}


def _beam(s):
    x, k = s["x"].float(), s["case"]["k"]
    b, w, v = x.shape
    total = s["cum"][:, :, None] + (x if s["lse"] is None else x - s["lse"][:, :, None])
    if s["mask"] is not None:
        total = torch.where(s["mask"], total, NEG_INF)
    total = total.view(b, w * v)
    # the order of (total, lowest place first) as whole numbers
    bits = (total + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    place = torch.topk((bits << 32) - torch.arange(w * v, device="cuda"), k, dim=1)[1]
    scores = total.gather(1, place)
    parents = place // v
    n = s["states"].shape[2]
    rows = torch.arange(b, device="cuda")[:, None]
    moved = s["states"][rows, parents]
    there = torch.arange(n, device="cuda") < s["len"][rows, parents][:, :, None]
    return {"scores": scores, "tokens": (place % v).to(torch.int32), "parents": parents.to(torch.int32),
            "next": torch.where(there[..., None], moved, torch.zeros_like(moved[:1, :1, :1]))}


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        taken = sum(_ceil(c + n, page) - _ceil(c, page) for c, n in zip(cached, new))
        return {"bytes": 16 * len(new) + case["pages"] / 8 + 8 * taken + 8 * sum(new), "flops": 0}
    if op == "append":
        return {"bytes": case["tokens"] * (8 + 8 * case["heads"] * case["dim"]), "flops": 0}
    if op == "attention":
        cached, new = _lengths(case)
        share = case["density"] * 0.96 + 0.02 if case["density"] < 1 else 1.0  # what passes, single slots included
        keys = sum(c + n for c, n in zip(cached, new)) * share
        pairs = sum(n * c + n * (n + 1) / 2 for c, n in zip(cached, new)) * share
        held = sum(_ceil(c + n, case["page"]) for c, n in zip(cached, new))
        listing = held * case["page"] / 8 + 4 * keys + 4 * sum(new) if case["density"] < 1 else 0
        return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + sum(new) * case["heads"] * (4 * case["dim"] + 4) +
                4 * held + listing, "flops": 4 * pairs * case["heads"] * case["dim"]}
    rows = case["batch"] * case["beams"]
    moved = case["batch"] * case["k"] * case["states"] / 2 * 4  # half of a state is in use, on average
    read = rows * case["vocab"] * (4 if case["dtype"] == "f32" else 2)
    return {"bytes": read + moved + 12 * case["batch"] * case["k"], "flops": 2 * rows * case["vocab"]}


def exact(case, seed):
    """The computed numbers in 64 bits, request by request; whole numbers and moved states have no such value."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        page = case["page"]
        for t, x in ((k, s["k"]), (v, s["v"])):
            t[s["slots"] // page, s["slots"] % page] = x.double()
        return {"k_cache": k, "v_cache": v}
    if case["op"] == "beam":
        x = s["x"].double()
        if s["lse"] is not None:
            x -= s["lse"].double()[:, :, None]
        x += s["cum"].double()[:, :, None]
        if s["mask"] is not None:
            x[:, :, ~s["mask"]] = NEG_INF
        best = torch.sort(torch.topk(x.flatten(1), case["k"], dim=1)[0], dim=1, descending=True)[0]
        return {"scores": best, "tokens": None, "parents": None, "next": None}
    page, kv_heads, group = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(s["lse"].shape, NEG_INF, device="cuda", dtype=torch.float64)
    kc = s["k_cache"].view(-1, kv_heads, case["dim"])
    vc = s["v_cache"].view(-1, kv_heads, case["dim"])
    cached, new = _lengths(case)
    at = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        here = torch.arange(c + n, device="cuda")
        slot = s["table"][r, here // page].long() * page + here % page
        if "visible" in s:
            here, slot = here[s["visible"][slot]], slot[s["visible"][slot]]
        for h in range(kv_heads if slot.numel() else 0):
            k, v = kc[slot, h].double(), vc[slot, h].double()
            for i in range(0, n, 4096):
                j = min(n, i + 4096)
                q = s["q"][at + i:at + j, h * group:(h + 1) * group].double()
                p = torch.einsum("tgd,kd->gtk", q, k) / math.sqrt(case["dim"])
                p.masked_fill_(here[None, None] > c + torch.arange(i, j, device="cuda")[None, :, None], NEG_INF)
                z = torch.logsumexp(p, 2)
                p = torch.exp(p - torch.where(z == NEG_INF, 0.0, z)[:, :, None])
                out[at + i:at + j, h * group:(h + 1) * group] = torch.einsum("gtk,kd->tgd", p, v)
                lse[at + i:at + j, h * group:(h + 1) * group] = z.t()
        at += n
    return {"out": out, "lse": lse, **({"sel": None, "sel_len": None, "limits": None} if "visible" in s else {})}
