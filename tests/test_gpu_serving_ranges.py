"""The serving operators at the ends of their values' ranges, and graphs whose calls have workspaces."""
import numpy as np
import pytest
import torch

from oracle import serving_oracle as O
from tensorrt_llm.quantization import group as G
from tensorrt_llm.runtime import paged_kv8 as P
from test_gpu_serving_ops import HALF, gpu, numbers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('rows,n', [(1, 40), (9, 100), (40, 300), (300, 300), (1500, 1100)])
def test_products_of_large_bfloat16(rows, n, group):
    """Values just below 2^113 are multiplied as any others, with the bound that the operator's other tests derive; a row of 2^126 is NaN or
    infinite, and no other one is."""
    rng = np.random.default_rng(rows + group)
    k = 416
    q = rng.integers(-8, 8, (n, k)).astype(np.int8)
    s = torch.from_numpy(rng.uniform(0.01, 0.2, (n, -(-k // group))).astype(np.float32)).bfloat16()
    x = torch.from_numpy((rng.uniform(1, 1.99, (rows, k)) * rng.choice([-1, 1], (rows, k))).astype(np.float32)).bfloat16() * 2.0**112
    f = G.GroupQuantMatmul(torch.from_numpy(q).cuda(), s.cuda(), group)
    y = f(x.cuda())
    want, terms, plain = O.group_product(x.float().numpy(), q, s.float().numpy(), group)
    bound = (k / 32 + 32) * 2.0**-24 * terms + HALF['bf16'] * np.abs(want) * 1.01 + 32 * 2.0**-24 * 280 * plain
    assert (np.abs(numbers(y) - want) <= bound).all(), float((np.abs(numbers(y) - want) / bound).max())
    if rows > 1:
        bad = x.clone()
        bad[1] *= 2.0**14
        got = f(bad.cuda())
        keep = [i for i in range(rows) if i != 1]
        assert not got[1].float().isfinite().any() and torch.equal(got[keep], y[keep])


def test_graphs_of_attention_with_workspaces():
    """Two graphs whose calls split their keys, replayed in turn and between eager calls of other sizes: the bits of eager calls."""
    torch.manual_seed(2)
    page, size, kv, heads = 64, 128, 2, 8
    cache = P.PagedKV8Cache(torch.randint(-127, 128, (120, 2, kv, page * size), dtype=torch.int8, device='cuda'), torch.rand((120, 2, kv), device='cuda') * 0.02, page, size)
    table = torch.randperm(120, device='cuda').int().view(2, 60)
    args = [(table[:1], gpu([0, 1]), gpu([3800]), 1), (table, gpu([0, 1, 40]), gpu([2900, 3500]), 39)]
    qs = [torch.randn((n, heads, size), device='cuda').half() for n in (1, 40)]
    graphs, outs = [], []
    for q, a in zip(qs, args):
        cache.attention(q, *a)  # what a first call sets up is there
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            outs.append(cache.attention(q, *a))
        torch.cuda.synchronize()
        graphs.append(g)
    for i in range(6):
        for q in qs:
            q.copy_(torch.randn_like(q))
        for g in graphs if i % 2 else graphs[::-1]:
            g.replay()
            torch.full((1 << 20, ), float('nan'), device='cuda').sum()
        for q, a, o in zip(qs, args, outs):
            assert torch.equal(cache.attention(q, *a), o)
