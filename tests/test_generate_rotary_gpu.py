"""The example with positions, norms of queries and keys, prompts by pieces and windows, against plain products and attention over whole sequences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(model, x):
    """Outputs of every token of one sequence x [tokens][hidden], in fp32 over the dense weights, rounded where the example rounds."""
    def norm(t, eps):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)

    def rotate(t, weight):  # [n][heads][d]
        t = norm(t, 1e-6) * weight.float()
        cos, sin = model.angles[:n].chunk(2, 1)
        a, b = t.chunk(2, -1)
        return torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], -1).half().float()
    x = x.float()
    n, heads, kv, d = len(x), model.heads, model.kv_heads, model.head_dim
    place = torch.arange(n, device="cuda")
    seen = place[None] <= place[:, None]
    if model.window is not None:
        seen &= (place[None] > place[:, None] - model.window) | (place[None] < model.sinks)
    for (qkv, out, up, down), (qw, kw) in zip(model.layers, model.head_norms):
        y = (norm(x, 1e-5).half().float() @ qkv.dense()).half().float().view(n, heads + 2 * kv, d)
        q, k = rotate(y[:, :heads], qw), rotate(y[:, heads:heads + kv], kw)
        o = torch.empty((n, heads, d), device="cuda")
        for h in range(heads):
            s = q[:, h] @ k[:, h // (heads // kv)].T / math.sqrt(d)
            o[:, h] = torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ y[:, heads + kv + h // (heads // kv)]
        x = (x + (o.half().float().view(n, -1) @ out.dense()).half().float()).half().float()
        x = (x + (torch.relu((norm(x, 1e-5).half().float() @ up.dense()).half().float()) @ down.dense()).half().float()).half().float()
    return norm(x, 1e-5)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("piece", [None, 64, 7])
def test_generate(hq, heads, kv_heads, head_dim, window, sinks, piece):
    from hecbench_amd.examples.generate import Decoder, Server
    model = Decoder(layers=2, heads=heads, kv_heads=kv_heads, head_dim=head_dim, hidden=512, wide=1024, seed=3, rotary=10000.0, longest=512,
                    window=window, sinks=sinks)
    gen = torch.Generator(device="cuda").manual_seed(4)
    prompts = [torch.randn((n, 512), generator=gen, device="cuda").half() for n in (33, 1, 150)]
    tokens, samples = 9, 2
    server = Server(model, prompts, samples, tokens)
    inputs, last = server.run(tokens, compact_every=4, piece=piece)
    assert server.cache.missing.item() == 0
    assert server.cache.lengths.tolist() == [len(p) + tokens for p in prompts for _ in range(samples)]
    # as without positions: about ten roundings of 2^-11 on the way to a token, in quadrature 2e-3 of the output's size, and two more for
    # rotated queries and keys; the bound is several times that
    for row in range(len(prompts) * samples):
        whole = torch.cat([prompts[row // samples]] + [x[row:row + 1] for x in inputs])
        want = plain(model, whole)[-1]
        err = (last[row].float() - want).norm() / want.norm()
        assert err <= 1e-2, (row, err.item())
