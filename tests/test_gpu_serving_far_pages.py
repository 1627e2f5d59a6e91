"""Attention over pages whose scales are far from each other, as an infinity among bfloat16 values leaves them: rows that do not see such a page do not
know of it, rows that do stay finite."""
import numpy as np
import pytest
import torch

from oracle import serving_oracle as O
from tensorrt_llm.runtime import paged_kv8 as P
from test_gpu_serving_ops import HALF, TYPES, gpu, numbers

pytestmark = pytest.mark.gpu
PAGE = 16


def cache_of(rng, pages, size, least=64):
    """int8 elements of magnitude `least` .. 127, so that every channel of a page has a part of its scale's size; scales of 0.01 .. 0.02."""
    bits = rng.integers(least, 128, (pages, 2, 1, PAGE * size)) * rng.choice([-1, 1], (pages, 2, 1, PAGE * size))
    pool = torch.from_numpy(bits.astype(np.int8)).cuda()
    return P.PagedKV8Cache(pool, gpu(rng.uniform(0.01, 0.02, (pages, 2, 1)), torch.float32), PAGE, size)


def check(cache, q, dtype, lens, rows, window=0, max_kv=None):
    """As the operator's other tests bound it: scores, weights (2^-11) and sums, then one rounding of the result."""
    size, table, at = cache.head_size, np.zeros((len(lens), -(-max(lens) // PAGE)), np.int32), 0
    for b, n in enumerate(lens):
        have = -(-n // PAGE)
        table[b, :have] = np.arange(at, at + have)
        at += have
    cu = np.concatenate([[0], np.cumsum(rows)])
    got = numbers(cache.attention(q.cuda(), gpu(table), gpu(cu), gpu(lens), max(rows), max_kv, window))
    want, spread, worst = O.attention(q.float().numpy(), cache.pool.cpu().float().numpy(), cache.scales.cpu().numpy(), table, cu, lens, PAGE, size**-0.5, window)
    z = (2 * size + 4) * 2.0**-24 * worst
    bound = (2 * z + 2.0**-11 + 2.0**-17) * spread * 1.01 + HALF[dtype] * np.abs(want) * 1.01 + 1e-30
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    return got


# (cached tokens, rows): tokens alone, split over workgroups, prompts, prompts split, both
SPANS = [([289], [3], None), ([4993], [2], 5000), ([300], [200], None), ([600], [90], 60000), ([700, 300], [2, 90], 30000)]


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', SPANS)
@pytest.mark.parametrize('far', [2.0**30, 2.0**100])
def test_a_page_behind_a_row_is_not_seen(lens, rows, max_kv, size, far):
    """The values' scale of the last request's last page is `far` times the others'.  Rows whose token stands in an earlier page have nothing of it, in the same
    tile of keys or of rows as others that have."""
    rng = np.random.default_rng(size)
    pages = [-(-n // PAGE) for n in lens]
    cache = cache_of(rng, sum(pages), size)
    cache.scales[-1, 1] *= far
    q = torch.from_numpy(rng.standard_normal((sum(rows), 2, size)).astype(np.float32)).bfloat16()
    got = check(cache, q, 'bf16', lens, rows, max_kv=max_kv)
    before = max(0, rows[-1] - ((lens[-1] - 1) % PAGE + 1))  # of the last request's rows
    assert (np.abs(got[sum(rows[:-1]):][:before]) < 3).all()


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', SPANS)
def test_a_page_before_the_window_is_not_seen(lens, rows, max_kv, size):
    rng = np.random.default_rng(size)
    window, pages = 40, [-(-n // PAGE) for n in lens]
    cache = cache_of(rng, sum(pages), size)
    first = lens[0] - rows[0] + 1 - window  # the first key that the first request's first row sees
    cache.scales[max(first, 0) // PAGE - 1, 1] *= 2.0**100
    q = torch.from_numpy(rng.standard_normal((sum(rows), 2, size)).astype(np.float32)).bfloat16()
    assert (np.abs(check(cache, q, 'bf16', lens, rows, window, max_kv)) < 3).all()


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', SPANS)
def test_a_far_page_without_weight_takes_nothing(lens, rows, max_kv, size):
    """A page of large values that every row sees and none weighs: its keys are against every query."""
    rng = np.random.default_rng(size + 1)
    pages = [-(-n // PAGE) for n in lens]
    cache = cache_of(rng, sum(pages), size)
    at = [sum(pages[:b]) for b in range(len(lens))]
    cache.pool[at, 0] = -100
    cache.scales[at, 0] = 0.25
    cache.scales[at, 1] = 2.0**40
    q = torch.from_numpy(rng.uniform(0.5, 1, (sum(rows), 2, size)).astype(np.float32)).bfloat16()  # scores of -100 and less
    assert (np.abs(check(cache, q, 'bf16', lens, rows, max_kv=max_kv)) < 3).all()


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', [([40], [1], None)] + SPANS)
def test_the_largest_values_stay_finite(lens, rows, max_kv, size):
    """Every value the largest that the cache gives bfloat16 (infinities count as it), then half of them its negative: the mean is exact but for the weights'
    rounding, and far from the type's end or within half a step of it."""
    rng = np.random.default_rng(size + 2)
    cache = cache_of(rng, sum(-(-n // PAGE) for n in lens), size)
    largest = float(torch.finfo(torch.bfloat16).max)
    cache.scales[:, 1] = largest / 127
    q = torch.zeros((sum(rows), 2, size), dtype=torch.bfloat16)
    for values in (torch.full((PAGE, ), 127), torch.tensor([127, -127] * (PAGE // 2))):
        cache.pool[:, 1] = values.to(torch.int8).cuda().repeat(size)
        check(cache, q, 'bf16', lens, rows, max_kv=max_kv)


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', SPANS)
def test_keys_of_nothing_in_a_page_of_the_largest(lens, rows, max_kv, size):
    """Keys that are zero under the largest scale score zero, however large the query."""
    rng = np.random.default_rng(size + 3)
    cache = cache_of(rng, sum(-(-n // PAGE) for n in lens), size)
    cache.pool[:, 0] = 0
    cache.scales[:, 0] = float(torch.finfo(torch.bfloat16).max) / 127
    q = torch.from_numpy(rng.standard_normal((sum(rows), 2, size)).astype(np.float32) * 2.0**20).bfloat16()
    check(cache, q, 'bf16', lens, rows, max_kv=max_kv)


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('lens,rows,max_kv', SPANS)
@pytest.mark.parametrize('loud', [2.0**8, 2.0**14])
def test_large_scores_that_are_equal(lens, rows, max_kv, size, loud):
    """Every key the same: weights are equal whatever the scores are (here up to some 2^22), and what rounding does to a score it does to the sum as well.  Off by the
    weights' rounding, the sums' and the result's."""
    rng = np.random.default_rng(size + 4)
    cache = cache_of(rng, sum(-(-n // PAGE) for n in lens), size)
    cache.pool[:, 0] = torch.from_numpy(rng.integers(64, 128, size).astype(np.int8)).cuda().repeat(PAGE)
    cache.scales[:, 0] = 0.0173
    cache.scales[:, 1] = 0.0119
    q = torch.from_numpy((rng.uniform(0.5, 1, (sum(rows), 2, size)) * rng.choice([-1, 1], (sum(rows), 2, 1)) * loud).astype(np.float32)).bfloat16()
    table, at = np.zeros((len(lens), -(-max(lens) // PAGE)), np.int32), 0
    for b, n in enumerate(lens):
        have = -(-n // PAGE)
        table[b, :have] = np.arange(at, at + have)
        at += have
    cu = np.concatenate([[0], np.cumsum(rows)])
    got = numbers(cache.attention(q.cuda(), gpu(table), gpu(cu), gpu(lens), max(rows), max_kv))
    want, spread, _ = O.attention(np.zeros(q.shape), cache.pool.cpu().float().numpy(), cache.scales.cpu().numpy(), table, cu, lens, PAGE, 1.0)
    assert (np.abs(got - want) <= (2.0**-11 + 2.0**-17) * spread * 1.01 + HALF['bf16'] * np.abs(want) * 1.01).all()
