"""A decoder of 3-bit weights that serves several requests at once: prompts taken in together, every request forked into samples
behind its prompt, tokens generated for all of them over one paged key / value cache, samples dropped, the cache compacted.

    python -m hecbench_amd.examples.generate [--layers N] [--prompts N] [--samples N] [--tokens N] [--piece N] [--window N] [--sinks N]

The weights are random and nothing is sampled: a token's embedding is what the last layer gave, so what is shown is how the operators
go together.  Every projection is hq.q3_gemm; what a step does to the cache is hq.cache_step (tables, forks, pages) once for all
layers.  In each layer, whole prompts go through hq.norm_rotate, hq.cache_write and hq.prompt_attention; the next tokens, or pieces of
prompts, through hq.cache_write_rotated and hq.paged_attention or, pieces and windows, hq.chunk_attention.
"""
import argparse
import time

import torch

import hecbench_amd as hq


class Linear:
    """GPTQ 3-bit weights [K][N]: codes, a scale and a zero point a column."""

    def __init__(self, k, n, gen):
        codes = torch.randint(0, 8, (k, n), dtype=torch.uint8, generator=gen, device="cuda")
        self.weight = hq.q3_pack(codes)
        self.scales = torch.full((n,), 0.6 / k ** 0.5, device="cuda")
        self.zeros = 3.5 * self.scales
        self.codes = codes

    def __call__(self, x):
        return hq.q3_gemm(x, self.weight, self.scales, self.zeros).half()

    def dense(self):  # for a check against a plain product
        return self.codes.float() * self.scales - self.zeros


def norm(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)).half()


class Decoder:
    """rotary: base of the positions' angles (None: no positions, and no norm of queries and keys), for up to `longest` tokens.  window: a token
    sees that many tokens up to itself (None: all of them) and the first `sinks`."""

    def __init__(self, layers=4, heads=32, kv_heads=8, head_dim=128, hidden=4096, wide=11008, seed=0, rotary=None, longest=8192, window=None, sinks=0):
        self.window, self.sinks = window, sinks
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.hidden = heads, kv_heads, head_dim, hidden
        rows = (heads + 2 * kv_heads) * head_dim
        self.layers = [(Linear(hidden, rows, gen), Linear(heads * head_dim, hidden, gen), Linear(hidden, wide, gen), Linear(wide, hidden, gen))
                       for _ in range(layers)]
        self.angles = None if rotary is None else hq.rotary_table(longest, head_dim, rotary)
        self.head_norms = [[(1 + 0.1 * torch.randn(head_dim, generator=gen, device="cuda")).half() for _ in range(2)]
                           for _ in range(layers if rotary is not None else 0)]

    def forward(self, x, attend):
        """x [tokens][hidden]; attend(layer, q, k, v) attends and keeps what it must."""
        for i, (qkv, out, up, down) in enumerate(self.layers):
            y = qkv(norm(x)).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            x = x + out(attend(i, q, k, v).reshape(-1, self.heads * self.head_dim))
            x = x + down(torch.relu(up(norm(x))))
        return norm(x)


class Cache:
    """The pages of all layers, and the tables of the requests that are under way."""

    def __init__(self, model, rows, pages, page=16, width=64):
        self.page, self.rows, self.model = page, rows, model
        self.pool = torch.zeros((2 * len(model.layers), pages, model.kv_heads, page, model.head_dim), dtype=torch.float16, device="cuda")
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.starts = self.missing = None

    def step(self, parent, add):
        """Row s goes on from row parent[s] (-1: empty) and gets room for add[s] tokens."""
        self.table, self.lengths, self.refs, self.starts, self.missing = hq.cache_step(
            self.pool, self.page, self.table, self.lengths, self.refs, parent, add)

    def compact(self):
        self.table, self.refs, live = hq.cache_compact(self.pool, self.table, self.refs)
        return live

    def pages(self, layer):
        return self.pool[2 * layer], self.pool[2 * layer + 1]

    def write(self, layer, q, k, v, cu):
        """Keys and values of the step's tokens; the queries, which go by the same positions."""
        if self.model.angles is None:
            hq.cache_write(k, v, *self.pages(layer), self.table, self.starts, cu)
            return q
        return hq.cache_write_rotated(q, k, v, *self.pages(layer), self.table, self.starts, cu, self.model.angles, *self.model.head_norms[layer])

    def attend(self, layer, q, cu):
        """Of the step's tokens, any number a row, to what is in the cache."""
        return hq.chunk_attention(q, *self.pages(layer), self.table, self.lengths, cu, window=self.model.window, sinks=self.model.sinks)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Server:
    def __init__(self, model, prompts, samples, tokens, page=16):
        """prompts: embeddings [tokens][hidden] of each; every one is continued `samples` times by `tokens` tokens."""
        self.model, self.samples = model, samples
        self.lengths = [len(p) for p in prompts]
        if model.angles is not None and max(self.lengths) + tokens > len(model.angles):
            raise ValueError(f"{max(self.lengths)} tokens and {tokens} more, and the model knows {len(model.angles)} positions")
        rows = len(prompts) * samples
        width = max(self.lengths) // page + tokens // page + 3
        # a prompt's pages once, and for every sample its tail, its tokens and a page to begin
        pages = sum(n // page + 1 for n in self.lengths) + rows * (tokens // page + 3)
        self.cache = Cache(model, rows, pages, page, width)
        self.prompts = torch.cat(prompts)
        self.groups = i32([i * samples for i in range(len(prompts) + 1)])
        self.shared = i32([n // page * page for n in self.lengths])  # whole pages stay shared behind a fork
        self.one_each = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
        self.same = torch.arange(rows, dtype=torch.int32, device="cuda")
        self.one = torch.ones(rows, dtype=torch.int32, device="cuda")

    def take_in(self, piece=None):
        """All prompts in one pass, or `piece` tokens of each at a time, into the first row of its samples; then the fork.  The prompts' last
        outputs, a row a sample."""
        n, s, c = len(self.lengths), self.samples, self.cache
        self.fork = i32([i // s * s for i in range(n * s)])  # every sample goes on from its prompt's row
        if piece:
            return self.take_in_pieces(piece)
        add, bounds, at = [0] * (n * s), [0], 0
        for i, length in enumerate(self.lengths):
            add[i * s] = length
            bounds += [at + length] * s
            at += length
        c.step(torch.full((n * s,), -1, dtype=torch.int32, device="cuda"), i32(add))
        cu, packed = i32(bounds), i32([0] + [b for b in bounds[1::s]])

        def attend(layer, q, k, v):
            if self.model.angles is not None:  # attention and the cache both take the keys
                q, k = hq.norm_rotate(q, k, self.model.angles, positions, *self.model.head_norms[layer])
            hq.cache_write(k, v, *c.pages(layer), c.table, c.starts, cu)
            return hq.prompt_attention(q, k, v, packed, window=self.model.window, sinks=self.model.sinks)

        positions = torch.cat([torch.arange(length, dtype=torch.int32, device="cuda") for length in self.lengths])
        x = self.model.forward(self.prompts, attend)
        last = x[packed[1:].long() - 1]
        return last.repeat_interleave(s, 0)

    def take_in_pieces(self, piece):
        n, s, c = len(self.lengths), self.samples, self.cache
        last = [None] * n
        begins = [sum(self.lengths[:i]) for i in range(n)]
        for done in range(0, max(self.lengths), piece):
            new = [max(0, min(piece, length - done)) for length in self.lengths]
            add, bounds = [0] * (n * s), [0]
            for i, m in enumerate(new):
                add[i * s] = m
                bounds += [bounds[-1] + m] * s
            cu = i32(bounds)
            c.step(self.same if done else torch.full((n * s,), -1, dtype=torch.int32, device="cuda"), i32(add))
            x = self.model.forward(torch.cat([self.prompts[b + done:b + done + m] for b, m in zip(begins, new)]),
                                   lambda layer, q, k, v: c.attend(layer, c.write(layer, q, k, v, cu), cu))
            for i, m in enumerate(new):
                if m and done + m == self.lengths[i]:
                    last[i] = x[bounds[(i + 1) * s] - 1]
        return torch.stack(last).repeat_interleave(s, 0)

    def token(self, x, parent, add=None):
        """The next token of every row: x [rows][hidden] in, its output back."""
        c = self.cache
        c.step(parent, self.one if add is None else add)

        def attend(layer, q, k, v):
            q = c.write(layer, q, k, v, self.one_each)
            if self.model.window is not None:
                return c.attend(layer, q, self.one_each)
            return hq.paged_attention(q, *c.pages(layer), c.table, c.lengths, self.groups, self.shared)

        return self.model.forward(x, attend)

    def run(self, tokens, compact_every=16, spread=0.02, piece=None):
        """Generates; the samples of a prompt are told apart by a little noise on their first embedding.  All inputs, [step][row][hidden]."""
        gen = torch.Generator(device="cuda").manual_seed(1)
        x = self.take_in(piece)
        x = x + (torch.randn(x.shape, generator=gen, device="cuda") * spread).half()
        inputs = []
        for i in range(tokens):
            inputs.append(x)
            x = self.token(x, self.same if i else self.fork)
            if i % compact_every == compact_every - 1:
                self.cache.compact()
        return inputs, x


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompts", type=int, default=4)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--piece", type=int, help="take prompts in by so many tokens each at a time")
    ap.add_argument("--window", type=int, help="tokens that a token sees, itself among them (default: all)")
    ap.add_argument("--sinks", type=int, default=0, help="first tokens that stay visible behind the window")
    a = ap.parse_args()
    hq.init()
    lengths = [200 + 173 * i for i in range(a.prompts)]
    model = Decoder(a.layers, rotary=10000.0, longest=max(lengths) + max(a.tokens, 2), window=a.window, sinks=a.sinks)
    gen = torch.Generator(device="cuda").manual_seed(2)
    prompts = [torch.randn((n, model.hidden), generator=gen, device="cuda").half() for n in lengths]
    Server(model, prompts, a.samples, 2).run(2, piece=a.piece)  # the first calls size the stream's workspace
    server = Server(model, prompts, a.samples, a.tokens)
    torch.cuda.synchronize()
    t = time.perf_counter()
    x = server.take_in(a.piece)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    for i in range(a.tokens):
        x = server.token(x, server.same if i else server.fork)
    live = server.cache.compact()
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    rows = a.prompts * a.samples
    assert server.cache.missing.item() == 0 and torch.isfinite(x).all()
    print("%d prompts, %d tokens: %.2f ms; %d samples, %d tokens each: %.2f ms a token of all; %d pages in use of %d" % (
        a.prompts, sum(server.lengths), (t1 - t) * 1e3, rows, a.tokens, (t2 - t1) * 1e3 / a.tokens, live.item(), server.cache.pool.shape[1]))


if __name__ == "__main__":
    main()
