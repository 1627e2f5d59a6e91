"""Batches at the ends of what the attention takes."""
import numpy as np
import pytest
import torch

from tensorrt_llm.runtime import paged_kv8 as P
from test_gpu_serving_ops import gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('at', [0, 4095])
def test_attention_of_a_prompt_beside_thousands_of_tokens(at):
    """4095 requests of a token and one of 8192 rows: more workgroups than a launch has in one dimension.  A token alone is its value; the prompt's rows are as in a
    call of their own (the same tiles: the weights' and results' roundings are the same or next to each other)."""
    torch.manual_seed(at)
    page, size, kv, heads, n, long = 16, 64, 8, 64, 4096, 8192
    pages = long // page
    cache = P.PagedKV8Cache(torch.randint(-127, 128, (n - 1 + pages, 2, kv, page * size), dtype=torch.int8, device='cuda'), torch.rand((n - 1 + pages, 2, kv), device='cuda') * 0.02, page, size)
    ids = torch.randperm(n - 1 + pages, device='cuda').int()
    table = torch.zeros((n, pages), dtype=torch.int32, device='cuda')
    others = [b for b in range(n) if b != at]
    table[others, 0] = ids[:n - 1]
    table[at] = ids[n - 1:]
    rows = [1] * n
    rows[at] = long
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = torch.randn((int(cu[-1]), heads, size), device='cuda').half()
    got = cache.attention(q, table, gpu(cu), gpu(rows), long, 100)
    first = cache.pool[ids[:n - 1].long(), 1].view(n - 1, kv, size, page)[..., 0].float() * cache.scales[ids[:n - 1].long(), 1][..., None]
    want = first.repeat_interleave(heads // kv, 1)
    mine = got[cu[:-1][others]].float()
    assert ((mine - want).abs() <= 2.0**-11 * 1.01 * want.abs() * 2 + 1e-7).all()  # the weight's rounding over its own, the result's
    alone = cache.attention(q[at:at + long], table[at:at + 1], gpu([0, long]), gpu([long]), long, 100)
    assert ((got[at:at + long].float() - alone.float()).abs() <= 2 * (2.0**-11 * alone.float().abs() + 2.0**-11 * 127 * 0.02)).all()
