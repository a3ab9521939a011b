"""A serving loop with drafted trees over a paged cache, on one GPU.

A toy one-layer model with random weights answers two prompts of different lengths, first one
token at a time, then with trees of drafted tokens of which some are right. Both ways give the
same tokens; the second takes fewer steps. It shows how the serving operators go together:

  paged_grow      room for the new tokens: cache blocks, slots
  gemm_epilogue   the projections
  rope_append     positions turned into q and k, keys and values written to the cache
  tree_attention  each new token over its request's context and its own branch
  adjust_logits   penalties for repeated tokens, a bias and a grammar mask
  paged_release   the blocks of rejected drafts go back

Run it with `python examples/serving_step.py` from the repository's root.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import matcoredsl_b200 as mcb  # noqa: E402

HEADS, KV_HEADS, DIM, VOCAB, BLOCK, BLOCKS, COLUMNS = 8, 2, 64, 1000, 16, 64, 16
WIDTH = HEADS * DIM


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Model:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[0] ** -0.5).bfloat16()  # noqa: E731
        self.embed = torch.randn(VOCAB, WIDTH, generator=g, device="cuda").bfloat16()
        self.w_qkv, self.w_o = w(WIDTH, (HEADS + 2 * KV_HEADS) * DIM), w(WIDTH, WIDTH)
        self.w_out = w(WIDTH, VOCAB)
        angle = (torch.arange(4096, device="cuda")[:, None]
                 * 10000.0 ** (-torch.arange(DIM // 2, device="cuda") / (DIM // 2)))
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1)


class Server:
    """Requests, their cache and their tokens. Every length stays on the GPU between the calls
    of a step; the host only reads the chosen tokens."""

    def __init__(self, model, prompts):
        self.model, self.tokens = model, [list(p) for p in prompts]
        self.prompt = [len(p) for p in prompts]
        n = len(prompts)
        self.table = torch.full((n, COLUMNS), -1, dtype=torch.int32, device="cuda")
        self.lens = ints([0] * n)
        self.free = torch.arange(BLOCKS, dtype=torch.int32, device="cuda")
        self.count = ints([BLOCKS])
        shape = (BLOCKS, BLOCK, KV_HEADS, DIM)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.grammar = torch.full((1, (VOCAB + 31) // 32), -1, dtype=torch.int32, device="cuda")
        self.grammar[0, 0] = ~0xFF  # the first eight tokens are never said
        self.steps = 0

    def forward(self, new, depths=None, mask=None, histories=None):
        """Logits of the new tokens of each request (lists), adjusted, as the most likely token of
        each row. `depths`: positions of drafted tokens relative to their request's length."""
        self.steps += 1
        m, flat = self.model, [t for r in new for t in r]
        slots, positions, cu, after, left = mcb.paged_grow(
            self.table, self.lens, ints([len(r) for r in new]), self.free, self.count, BLOCK,
            tokens=len(flat))
        if depths is not None:  # a draft's position is its depth in the tree, not its place
            start = torch.repeat_interleave(self.lens, ints([len(r) for r in new]).long())
            positions = start + ints([d for r in depths for d in r])
        x = m.embed[ints(flat).long()]
        qkv = mcb.gemm_epilogue(x, m.w_qkv, out_dtype="bf16")
        q, k, v = (y.unflatten(1, (-1, DIM)) for y in qkv.split(
            [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1))
        q = mcb.rope_append(q, k, v, m.cos_sin, positions, slots, self.k, self.v)
        o = mcb.tree_attention(q, self.k, self.v, self.table, cu, after, mask)
        y = mcb.residual_rmsnorm(x, mcb.gemm_epilogue(o.flatten(1), m.w_o, out_dtype="bf16"))
        logits = mcb.gemm_epilogue(y, m.w_out, out_dtype="f32")
        # Each row is penalised for its own request's tokens and its own branch.
        rows = histories or [r[:i + 1] for r in new for i in range(len(r))]
        full = [self.tokens[b] + list(h) for b, h in zip(
            (b for b, r in enumerate(new) for _ in r), rows)]
        starts = [0]
        for h in full:
            starts.append(starts[-1] + len(h))
        prompt = [self.prompt[b] for b, r in enumerate(new) for _ in r]
        one = torch.ones(len(flat), device="cuda")
        mcb.adjust_logits(logits, ints([t for h in full for t in h]), ints(starts), ints(prompt),
                          repetition=1.2 * one, presence=0.1 * one, frequency=0.05 * one,
                          bias_ids=ints([3] * len(flat)), bias_values=-2.0 * one,
                          bias_cu=ints(range(len(flat) + 1)),
                          allowed=self.grammar.expand(len(flat), -1).contiguous(), out=logits)
        self.slots, self.after, self.left = slots, after, left
        return logits.argmax(1).tolist()

    def keep(self, kept):
        """Takes the drafts of the last step back, but for those in `kept` (places among each
        request's new tokens, in order), whose cache rows move to the front."""
        first = 0
        flat_k, flat_v = self.k.view(-1, KV_HEADS, DIM), self.v.view(-1, KV_HEADS, DIM)
        lens = self.lens.tolist()
        for b, (places, n) in enumerate(kept):
            src = self.slots[first:first + n][ints(places).long()].long()
            dst = self.slots[first:first + len(places)].long()
            flat_k[dst], flat_v[dst] = flat_k[src].clone(), flat_v[src].clone()
            lens[b] += len(places)
            first += n
        self.lens = ints(lens)
        self.count = mcb.paged_release(self.table, self.after, self.lens, self.free, self.left,
                                       BLOCK)


def answer(model, prompts, count):
    """`count` tokens for each prompt, one at a time."""
    s = Server(model, prompts)
    # the prompts themselves: every row's history is what stands before it
    tokens, s.tokens = s.tokens, [[] for _ in prompts]
    rows = s.forward(tokens)
    s.tokens = tokens
    s.keep([(range(len(t)), len(t)) for t in tokens])
    ends = [sum(len(t) for t in tokens[:b + 1]) - 1 for b in range(len(tokens))]
    chosen = [rows[e] for e in ends]
    for _ in range(count - 1):
        rows = s.forward([[c] for c in chosen])
        s.keep([([0], 1) for _ in chosen])
        for b, c in enumerate(chosen):
            s.tokens[b].append(c)
        chosen = rows
    return [t + [c] for t, c in zip(s.tokens, chosen)], s


def answer_with_drafts(model, prompts, known, count):
    """The same with trees of drafts: a chain of four guesses and, beside each, a wrong one. The
    guesses are taken from `known` (what a drafter would say), every third of them spoilt."""
    s = Server(model, prompts)
    tokens, s.tokens = s.tokens, [[] for _ in prompts]
    rows = s.forward(tokens)
    s.tokens = tokens
    s.keep([(range(len(t)), len(t)) for t in tokens])
    ends = [sum(len(t) for t in tokens[:b + 1]) - 1 for b in range(len(tokens))]
    chosen = [rows[e] for e in ends]  # decided, not yet in the cache
    goal = [len(p) + count for p in prompts]
    while any(len(t) + 1 < g for t, g in zip(s.tokens, goal)):
        new, depths, histories, bits, parents = [], [], [], [], []
        for b, c in enumerate(chosen):
            have = len(s.tokens[b])
            tree, depth, paths, parent = [c], [0], [[c]], [-1]
            last = 0
            for d in range(1, 5):
                guess = known[b][have + d] if have + d < len(known[b]) else 0
                if (have + d) % 3 == 0:
                    guess = (guess + 1) % VOCAB
                for t in (guess, (guess + 7) % VOCAB):
                    tree.append(t)
                    depth.append(d)
                    parent.append(last)
                    paths.append(paths[last] + [t])
                last = len(tree) - 2  # the guess carries the chain on
            new.append(tree)
            depths.append(depth)
            histories += paths
            parents.append(parent)
            for i in range(len(tree)):
                row, j = 0, i
                while j >= 0:
                    row, j = row | 1 << j, parent[j]
                bits.append([row])
        rows = s.forward(new, depths, ints(bits), histories)
        kept, first = [], 0
        for b, tree in enumerate(new):
            at, path = 0, [0]
            while True:  # follow the model's own choice as long as it was drafted
                choice = rows[first + at]
                child = [i for i in range(len(tree)) if parents[b][i] == at and tree[i] == choice]
                if not child or len(s.tokens[b]) + len(path) + 1 >= goal[b]:
                    break
                at = child[0]
                path.append(at)
            if len(s.tokens[b]) + 1 >= goal[b]:
                path = []  # this request is done: nothing of the step counts
            kept.append((path, len(tree)))
            if path:
                s.tokens[b] += [tree[i] for i in path]
                chosen[b] = rows[first + at]
            first += len(tree)
        s.keep(kept)
    return [t + [c] for t, c in zip(s.tokens, chosen)], s


def main():
    model = Model()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (37, 5)]
    plain, one = answer(model, prompts, 24)
    drafted, many = answer_with_drafts(model, prompts, plain, 24)
    same = plain == drafted
    print(f"one token at a time: {one.steps} steps; with drafted trees: {many.steps} steps; "
          f"the same tokens: {same}")
    return same, one, many


if __name__ == "__main__":
    sys.exit(0 if main()[0] else 1)
