"""Constrained beam search over a paged cache, with bitmaps for everything that is a set.

A small decoder with random weights answers several prompts of different lengths at once:

  * the cache's free pages are a bitmap: `paged_plan` takes pages from it, and whatever no beam holds any
    more goes back to it with a set operation;
  * the slots of prompt tokens that nobody may look at (a redacted passage, say) are a bitmap:
    `paged_select` lists the rest once a step, and every layer's `paged_attention` reads that list;
  * the tokens that an answer may use are a bitmap, which `beam_select` reads as it lies.

A page holds one token here, so beams share their past by sharing pages: after `beam_select`, `beam_reorder`
moves the rows of the block tables and no key or value is copied.

    python cu-roaring-bitmap_amd/examples/serving.py --prompts 3 --beams 4 --tokens 16
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "python"))
import curoaring as cr  # noqa: E402


class Decoder:
    """Weights of a small decoder: `layers` of attention with shared key heads and a two-layer perceptron."""

    def __init__(self, vocab=2000, layers=2, heads=8, kv_heads=2, dim=64, positions=512, dtype=torch.float16, seed=0):
        g = torch.Generator(device="cpu").manual_seed(seed)
        wide = heads * dim

        def weight(*shape):
            return (torch.randn(shape, generator=g) * shape[0] ** -0.5).to("cuda", dtype)

        self.heads, self.kv_heads, self.dim, self.vocab, self.dtype = heads, kv_heads, dim, vocab, dtype
        self.embed = torch.randn((vocab, wide), generator=g).to("cuda", dtype)
        self.places = torch.randn((positions, wide), generator=g).to("cuda", dtype)
        self.out = weight(wide, vocab)
        self.layers = [dict(q=weight(wide, wide), k=weight(wide, kv_heads * dim), v=weight(wide, kv_heads * dim),
                            o=weight(wide, wide), up=weight(wide, 2 * wide), down=weight(2 * wide, wide))
                       for _ in range(layers)]

    @staticmethod
    def norm(x):
        return torch.nn.functional.layer_norm(x.float(), x.shape[-1:]).to(x.dtype)

    def forward(self, tokens, positions, attend):
        """Logits (float32) of the tokens; `attend(layer, q, k, v)` is the attention over what came before."""
        x = self.embed[tokens] + self.places[positions]
        for i, w in enumerate(self.layers):
            y = self.norm(x)
            o = attend(i, (y @ w["q"]).view(-1, self.heads, self.dim), (y @ w["k"]).view(-1, self.kv_heads, self.dim),
                       (y @ w["v"]).view(-1, self.kv_heads, self.dim))
            x = x + o.flatten(1) @ w["o"]
            x = x + torch.relu(self.norm(x) @ w["up"]) @ w["down"]
        return self.norm(x).float() @ self.out.float()


class Server:
    """A paged cache of `pages` tokens for one decoder, and the sets that go with it."""

    def __init__(self, model, pages=4096):
        self.model, self.pages = model, pages
        shape = (len(model.layers), pages, 1, model.kv_heads, model.dim)
        self.k = torch.empty(shape, dtype=model.dtype, device="cuda")
        self.v = torch.empty(shape, dtype=model.dtype, device="cuda")
        self.all = cr.upload_from_device_ids(torch.arange(pages, dtype=torch.int32, device="cuda"), pages)
        self.free = cr.deep_copy(self.all)
        self.visible = cr.deep_copy(self.all)

    def close(self):
        for g in (self.all, self.free, self.visible):
            cr.free(g)

    def without(self, d_ids):
        """Every page or slot but these (one slot a page: their numbers are the same)."""
        ids = cr.upload_from_device_ids(torch.unique(d_ids[d_ids >= 0]).to(torch.int32), self.pages)
        rest = cr.set_operation(self.all, ids, cr.ANDNOT)
        cr.free(ids)
        return rest

    def hide(self, d_slots):
        cr.free(self.visible)
        self.visible = self.without(d_slots)

    def plan(self, table, cached, new, n_tokens):
        """Pages and slots for `new` more tokens a row; the pages are in use until keep_only() says otherwise."""
        def ints(n):
            return torch.empty(n, dtype=torch.int32, device="cuda")

        rows = cached.numel()
        slots, starts, kv_len = torch.empty(n_tokens, dtype=torch.int64, device="cuda"), ints(rows + 1), ints(rows)
        taken, counts = ints(n_tokens), ints(3)
        cr.paged_plan(self.free, self.pages, 1, cached, new, table, slots, starts, kv_len, taken, counts)
        if int(counts[2]):
            raise RuntimeError(f"the cache is full: {int(counts[2])} pages are missing")
        return slots, starts, kv_len

    def keep_only(self, table, length):
        """Pages that none of the rows holds any more are free again."""
        held = torch.arange(table.shape[1], device="cuda")[None, :] < length[:, None]
        cr.free(self.free)
        self.free = self.without(table[held])

    def step(self, tokens, table, slots, starts, kv_len, max_new, max_kv):
        """Logits [rows, vocab] after each row's last new token."""
        rows, cols = table.shape
        sel = torch.empty((rows, cols), dtype=torch.int32, device="cuda")
        sel_len = torch.empty(rows, dtype=torch.int32, device="cuda")
        limits = torch.empty(tokens.numel(), dtype=torch.int32, device="cuda")
        cr.paged_select(self.visible, table, starts, kv_len, 1, sel, sel_len, limits)

        def attend(layer, q, k, v):
            out = torch.empty_like(q)
            cr.paged_append(k, v, slots, self.k[layer], self.v[layer])
            cr.paged_attention(q, self.k[layer], self.v[layer], table, starts, kv_len, out,
                               selection=(sel, sel_len, limits), max_new=max_new, max_kv=max_kv)
            return out

        new = (starts[1:] - starts[:-1]).long()
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), new, output_size=tokens.numel())
        place = torch.arange(tokens.numel(), device="cuda") - starts[1:].long()[row] + kv_len.long()[row]
        logits = self.model.forward(tokens, place, attend)
        return logits[starts[1:].long() - 1]


def generate(server, prompts, hidden, allowed, beams=4, n_tokens=16):
    """The `beams` best answers of n_tokens tokens to each prompt: tokens [B, beams, n_tokens], log-probabilities.

    prompts: lists of token ids, none empty.  hidden: for each, which of its tokens the rest may not look at.
    allowed: a bitmap of the tokens that an answer may use, of at least `beams` of them."""
    batch, model = len(prompts), server.model
    lengths = [len(p) for p in prompts]
    cols = max(lengths) + n_tokens

    def select(logits, cum):
        """Continuations [B, beams] of the beams, by the sum of their log-probabilities."""
        scores = torch.empty((batch, beams), dtype=torch.float32, device="cuda")
        token, parent = (torch.empty((batch, beams), dtype=torch.int32, device="cuda") for _ in range(2))
        lse = torch.logsumexp(logits, -1).view(batch, -1)
        cr.beam_select(logits.view(batch, -1, model.vocab), cum, scores, token, parent, d_lse=lse, allowed=allowed)
        return scores, token, parent

    def moved(state, parent):
        to = torch.empty((batch, beams) + tuple(state.shape[2:]), dtype=state.dtype, device="cuda")
        cr.beam_reorder(state, parent, to)
        return to

    # the prompts, all at once
    table = torch.full((batch, cols), -1, dtype=torch.int32, device="cuda")
    new = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    slots, starts, kv_len = server.plan(table, torch.zeros_like(new), new, sum(lengths))
    mask = torch.tensor([bool(h) for row in hidden for h in row], device="cuda")
    server.hide(slots[mask])
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    logits = server.step(tokens, table, slots, starts, kv_len, max(lengths), max(lengths))
    scores, token, parent = select(logits, torch.zeros((batch, 1), device="cuda"))
    table = moved(table.view(batch, 1, cols), parent)
    answer = torch.full((batch, beams, n_tokens), -1, dtype=torch.int32, device="cuda")
    answer[:, :, 0] = token
    length = new.view(batch, 1).expand(batch, beams).reshape(-1).contiguous()
    one = torch.ones_like(length)

    # one token of every beam at a time
    for i in range(1, n_tokens):
        rows = table.view(batch * beams, cols)
        server.keep_only(rows, length)
        slots, starts, kv_len = server.plan(rows, length, one, batch * beams)
        logits = server.step(token.view(-1).long(), rows, slots, starts, kv_len, 1, max(lengths) + i)
        length = kv_len
        scores, token, parent = select(logits, scores)
        table, answer = moved(table, parent), moved(answer, parent)
        answer[:, :, i] = token
    server.keep_only(table.view(batch * beams, cols), torch.zeros_like(length))
    return answer, scores


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=16)
    args = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    model = Decoder()
    server = Server(model)
    prompts = [torch.randint(0, model.vocab, (int(n),), generator=g).tolist()
               for n in torch.randint(1, 200, (args.prompts,), generator=g)]
    hidden = [[i % 5 == 3 for i in range(len(p))] for p in prompts]
    ids = torch.arange(0, model.vocab, 3, dtype=torch.int32, device="cuda")
    allowed = cr.upload_from_device_ids(ids, model.vocab)
    answer, scores = generate(server, prompts, hidden, allowed, args.beams, args.tokens)
    for b, prompt in enumerate(prompts):
        print(f"prompt {b} ({len(prompt)} tokens, {sum(hidden[b])} hidden)")
        for w in range(args.beams):
            print(f"  {float(scores[b, w]):9.3f}  {answer[b, w].tolist()}")
    cr.free(allowed)
    server.close()


if __name__ == "__main__":
    main()
