"""The operators of a quantised serving step (include/tllm_serving_api.h) through their Python entry points, against oracle/serving_oracle.py: page
plans and the cache's bits exactly, attention and 4-bit products within bounds that follow from their arithmetic (next to each assert)."""
import copy
import pickle

import numpy as np
import pytest
import torch

from oracle import serving_oracle as O
from tensorrt_llm.quantization import group as G
from tensorrt_llm.runtime import paged_kv8 as P

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}
HALF = {'fp16': 2.0**-11, 'bf16': 2.0**-8}  # a rounding to the type, relative
CACHE = {'int8': torch.int8, 'fp8': torch.float8_e4m3fn}


def gpu(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(dtype).cuda()


def numbers(t):
    return t.float().cpu().numpy()


# ------------------------------------------------------------------------------------------------ plan
def random_state(rng, n, page, wide, longest):
    """Requests with tables in a shuffled pool, the rest of the blocks in a ring that starts anywhere."""
    lens = rng.integers(0, longest + 1, n)
    have = -(-lens // page)
    blocks = int(have.sum()) + n * 3 + 5
    ids = rng.permutation(blocks)
    table, at = np.full((n, wide), -7, np.int32), 0
    for b in range(n):
        table[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    ring, head = np.full(blocks, -9, np.int32), int(rng.integers(blocks))
    ring[(head + np.arange(blocks - at)) % blocks] = ids[at:]
    return lens, ring, [head, blocks - at], table


def check_plan(lens, new, ring, state, table, page, n_rows, in_place=False, pad=0):
    want = O.plan(lens, new, ring, state, table, page, n_rows)
    wide = torch.full((table.shape[0], table.shape[1] + pad), -5, dtype=torch.int32, device='cuda')
    wide[:, :table.shape[1]] = gpu(table)
    t, r, l, s = wide[:, :table.shape[1]], gpu(ring), gpu(lens), gpu(state)
    out = P.StepPlan(len(lens), n_rows, 'cuda', lens=l if in_place else None, ring_state=s if in_place else None)
    P.plan_step(l, gpu(new), r, s, t, page, n_rows, out)
    for name, got in dict(lens=out.lens, cu=out.cu_tokens, slots=out.slot_map, places=out.positions, ring=r, state=out.ring_state, table=t).items():
        np.testing.assert_array_equal(got.cpu().numpy(), want[name], err_msg=name)
    assert int(out.status) == want['status']
    assert (wide[:, table.shape[1]:] == -5).all()
    return want


@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('n,page,longest,most', [(1, 64, 0, 1), (1, 16, 100, 1000), (7, 32, 90, 40), (64, 64, 700, 1), (300, 16, 60, 30), (4096, 128, 300, 2), (33, 64, 64, 3000), (4096, 128, 300, 127)])
def test_plan(n, page, longest, most, in_place):
    rng = np.random.default_rng(n * 131 + page)
    wide = -(-(longest + most) // page) + 1
    lens, ring, state, table = random_state(rng, n, page, wide, longest)
    new = rng.integers(-1, most + 1, n)
    need = int(sum(max(x, 0) for x in new))
    room, have = state[1], -(-lens // page)
    for b in range(n):  # what the ring does not have is not asked for
        take = -(-(lens[b] + max(new[b], 0)) // page) - have[b]
        if take > room:
            need -= new[b]
            new[b] = 0
        else:
            room -= take
    assert check_plan(lens, new, ring, state, table, page, need + 5, in_place, pad=3)['status'] == 0
    if need:
        check_plan(lens, new, ring, state, table, page, need, in_place)


def test_plan_on_page_borders():
    for length in (0, 15, 16, 17, 31, 32):
        for add in (-1, 0, 1, 15, 16, 17):
            lens = [length, 5, length]
            have = [-(-x // 16) for x in lens]
            table, ids = np.zeros((3, 5), np.int32), iter(range(100))
            for b in range(3):
                table[b, :have[b]] = [next(ids) for _ in range(have[b])]
            used = sum(have)
            ring = np.concatenate([np.arange(used, 20), np.zeros(used, int)])
            assert check_plan(lens, [add, 1, add], ring, [0, 20 - used], table, 16, 40)['status'] == 0


@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('rows', [20, 3000])
@pytest.mark.parametrize('what', ['table', 'ring', 'rows', 'length', 'count', 'head', 'huge', 'given'])
def test_plan_that_does_not_fit_changes_nothing(what, rows, in_place):
    lens, new, state = [3, 16, 40], [1, 1, 1], [2, 4]
    table, ring = np.array([[0, 0, 0], [1, 0, 0], [2, 3, 4]]), np.array([0, 0, 5, 6, 7, 8, 9, 0, 0, 0])
    if what == 'table':
        new = [1, 1, 9]
    elif what == 'ring':
        new, state = [14, 1, 1], [2, 1]
    elif what == 'rows':
        rows = 2
    elif what == 'length':
        lens = [3, -2, 40]
    elif what == 'count':
        state = [2, -1]
    elif what == 'head':
        state = [10, 4]
    elif what == 'huge':
        new = [2**31 - 1, 2**31 - 1, 2**31 - 1]
    elif what == 'given':
        new, state = [1, 1, -1], [2, 8]
    want = check_plan(lens, new, ring, state, table, 16, rows, in_place)
    assert want['status'] != 0 and set(want['slots']) <= {-1}


def test_plan_step_by_step_gives_blocks_back():
    """Requests come, grow and end over a pool that would not hold them all at once; the tables never share a block."""
    rng = np.random.default_rng(5)
    pool = P.DeviceBlockPool(40, 16, 6, 12)
    lens, ring, state, table = np.zeros(6, int), np.arange(40), [0, 40], np.zeros((6, 12), int)
    for step in range(60):
        new = np.where(rng.random(6) < 0.2, -1, rng.integers(0, 25, 6))
        out = pool.plan(gpu(new), 160)
        want = O.plan(lens, new, ring, state, table, 16, 160)
        assert int(out.status) == want['status']
        lens, ring, state, table = want['lens'], want['ring'], want['state'], want['table']
        np.testing.assert_array_equal(pool.lens.cpu().numpy(), lens)
        np.testing.assert_array_equal(pool.ring_state.cpu().numpy(), state)
        np.testing.assert_array_equal(pool.block_table.cpu().numpy(), table)
        np.testing.assert_array_equal(out.slot_map.cpu().numpy(), want['slots'])
        held = [table[b, j] for b in range(6) for j in range(-(-lens[b] // 16))]
        assert len(set(held)) == len(held) and len(held) + state[1] == 40


# ------------------------------------------------------------------------------------------------ append
class Cache:
    """A cache on the GPU and the oracle's image of it."""

    def __init__(self, rng, blocks, page, heads, size, kind, garbage=False):
        self.page, self.kind = page, kind
        bits = rng.integers(0, 256, (blocks, 2, heads, page * size), dtype=np.uint8)
        if kind == 'fp8' and not garbage:
            bits = np.where((bits & 0x7f) == 0x7f, bits ^ 1, bits)
        self.gpu = P.PagedKV8Cache(torch.from_numpy(bits).cuda().view(CACHE[kind]), gpu(rng.uniform(0.001, 0.02, (blocks, 2, heads)), torch.float32), page, size)
        self.pool, self.scales = numbers(self.gpu.pool), self.gpu.scales.cpu().numpy()

    def same(self):
        np.testing.assert_array_equal(self.gpu.scales.cpu().numpy(), self.scales)
        np.testing.assert_array_equal(numbers(self.gpu.pool), self.pool)


def values(rng, shape, dtype):
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * rng.choice([0.5, 4.0], shape[-1])).to(TYPES[dtype])
    return x, x.float().numpy()


def slots_of(rng, spans, page, blocks):
    """Rows of requests [(first position, rows)] in pages in any order -> slots, positions."""
    ids, slots, places, at = rng.permutation(blocks), [], [], 0
    for first, n in spans:
        pages = -(-(first + n) // page)
        own = ids[at:at + pages]
        at += pages
        assert at <= blocks
        places += list(range(first, first + n))
        slots += [int(own[t // page]) * page + t % page for t in range(first, first + n)]
    return np.array(slots, np.int64), np.array(places)


SPANS = [[(0, 1)], [(5, 1)], [(0, 16), (7, 1), (63, 2)], [(3, 150), (0, 1), (130, 3), (15, 1), (16, 1)], [(i * 7 % 130, 1) for i in range(70)], [(1, 700)]]


@pytest.mark.parametrize('dtype,kind', [('fp16', 'int8'), ('bf16', 'fp8'), ('bf16', 'int8'), ('fp16', 'fp8')])
@pytest.mark.parametrize('spans', SPANS)
@pytest.mark.parametrize('page,size,heads', [(64, 128, 3), (16, 64, 2), (128, 256, 1), (32, 128, 5), (16, 256, 1), (128, 64, 2)])
def test_append_to_the_bit(page, size, heads, spans, dtype, kind):
    rng = np.random.default_rng(page * size + heads + len(spans))
    blocks = sum(-(-(a + n) // page) for a, n in spans) + 2
    c = Cache(rng, blocks, page, heads, size, kind)
    slots, _ = slots_of(rng, spans, page, blocks)
    k, kf = values(rng, (len(slots), heads, size), dtype)
    v, vf = values(rng, (len(slots), heads, size), dtype)
    c.gpu.append(k.cuda(), v.cuda(), gpu(slots))
    O.append(c.pool, c.scales, kf, vf, slots, page, kind, torch.finfo(TYPES[dtype]).max)
    c.same()


@pytest.mark.parametrize('spans', [[(5, 1100)], [(i, 1) for i in range(300)] + [(0, 900)], [(100, 3000), (0, 1), (31, 1), (63, 2), (0, 1300)], [(40, 70000)]], ids=['one', 'tokens', 'prompts', 'most'])
def test_append_of_many_rows(spans):
    """Workgroups that look for runs in 16 rows, and in a page of rows."""
    rng = np.random.default_rng(len(spans))
    page, size, heads, blocks = 32, 64, 8, sum(-(-(a + n) // 32) for a, n in spans)
    c = Cache(rng, blocks, page, heads, size, 'int8')
    slots, _ = slots_of(rng, spans, page, blocks)
    k, kf = values(rng, (len(slots), heads, size), 'fp16')
    v, vf = values(rng, (len(slots), heads, size), 'fp16')
    c.gpu.append(k.cuda(), v.cuda(), gpu(slots))
    O.append(c.pool, c.scales, kf, vf, slots, page, 'int8', 65504)
    c.same()


def test_append_and_attention_beyond_32_bits():
    """A pool of more than 2^32 bytes: pages at its end hold and give back what pages at the beginning of a small one do."""
    rng = np.random.default_rng(6)
    page, size, heads, n = 128, 128, 8, 17500  # 4.6 GB
    far = P.PagedKV8Cache(torch.empty((n, 2, heads, page * size), dtype=torch.int8, device='cuda'), torch.zeros((n, 2, heads), device='cuda'), page, size)
    near = P.PagedKV8Cache.empty(4, page, heads, size)
    assert far.pool.numel() > 2**32
    x = torch.from_numpy(rng.standard_normal((300, 3 * heads, size)).astype(np.float32)).half().cuda()
    at = np.arange(300)
    outs = []
    for cache, ids in ((near, [2, 0, 3]), (far, [n - 1, n - 3, n - 2])):
        slots = gpu([ids[t // page] * page + t % page for t in at])
        cache.append(x[:, heads:2 * heads], x[:, 2 * heads:], slots)
        table = gpu([ids])
        outs.append([cache.attention(x[:, :heads], table, gpu([0, 300]), gpu([300]), 300), cache.attention(x[:1, :heads], table, gpu([0, 1]), gpu([290]), 1),
                     cache.pool[ids[0]], cache.pool[ids[1]], cache.scales[ids[:2]]])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize('dtype,kind,pairs', [('fp16', 'int8', False), ('bf16', 'fp8', True), ('fp16', 'fp8', False), ('bf16', 'int8', True)])
@pytest.mark.parametrize('size,rot,q_heads', [(64, 64, 8), (128, 128, 4), (128, 32, 5), (256, 240, 2), (256, 16, 3)])
def test_append_rotates(size, rot, q_heads, dtype, kind, pairs):
    """Views into one packed projection, rows that are passed over in between, queries in place."""
    rng = np.random.default_rng(size + rot)
    page, heads, spans = 32, 2, [(900, 70), (40000, 2), (0, 33)]
    places = np.concatenate([np.arange(a, a + n) for a, n in spans])
    blocks, n = 12, len(places) + 2
    own = rng.permutation(blocks)  # pages in the order that the rows come to them: only the part of a request near its end is held
    slots, at = [], -1
    for a, m in spans:
        for t in range(a, a + m):
            at += t % page == 0 or t == a
            slots.append(int(own[at]) * page + t % page)
    slots = np.array(slots[:70] + [-1] + slots[70:] + [-1])  # between two requests and at the end: a page's rows are consecutive
    places = np.concatenate([places[:70], [-1], places[70:], [7]])
    c = Cache(rng, blocks, page, heads, size, kind)
    qkv, f = values(rng, (n, q_heads + 2 * heads, size), dtype)
    rope = P.rope_table(41000, rot)
    turned = O.rotate(f, rope.cpu().numpy()[places], pairs)
    O.append(c.pool, c.scales, turned[:, q_heads:q_heads + heads], f[:, q_heads + heads:], slots, page, kind, torch.finfo(TYPES[dtype]).max)
    x = qkv.cuda()
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    fresh = c.gpu.append(k, v, gpu(slots), gpu(places), rope, q, rope_pairs=pairs)
    c.same()
    live = slots >= 0
    want = torch.from_numpy(turned[:, :q_heads]).to(TYPES[dtype])
    assert torch.equal(fresh.cpu()[live], want[live])
    # against 64 bits: three fp32 roundings of the products and the sum (2^-24 of each term), one to the type
    exact = O.rotate(f[:, :q_heads].astype(np.float64), rope.cpu().numpy()[places].astype(np.float64), pairs)
    size_of = np.abs(f[:, :q_heads]).max() * 2 * 3 * 2.0**-24
    assert (np.abs(numbers(fresh) - exact)[live] <= (HALF[dtype] * np.abs(exact) * 1.001 + size_of + 1e-8)[live]).all()
    back = c.gpu.append(k, v, gpu(slots), gpu(places), rope, q, q_out=q, rope_pairs=pairs)
    assert back.data_ptr() == x.data_ptr() and torch.equal(q.cpu()[live], want[live]) and torch.equal(q.cpu()[~live], qkv[~live][:, :q_heads])


@pytest.mark.parametrize('kind', ['int8', 'fp8'])
def test_append_token_by_token_grows_the_scale(kind):
    """Rising magnitudes: every token brings what is held to a larger scale.  Each stored value is within the sum of its roundings: half a step of every
    scale it went through (e4m3: 2^-4 of the value, or half of its smallest step)."""
    rng = np.random.default_rng(3)
    page, size, heads = 16, 64, 2
    c = Cache(rng, 3, page, heads, size, kind, garbage=True)
    x = rng.standard_normal((page, heads, size)).astype(np.float32) * (1.3**np.arange(page))[:, None, None].astype(np.float32)
    t = torch.from_numpy(x).half()
    x = t.float().numpy()
    steps = np.zeros((page, heads))
    for i in range(page):
        s = gpu([16 + i])
        c.gpu.append(t[i:i + 1].cuda(), t[i:i + 1].cuda(), s)
        O.append(c.pool, c.scales, x[i:i + 1], x[i:i + 1], [16 + i], page, kind, 65504)
        np.testing.assert_array_equal(c.gpu.scales.cpu().numpy(), c.scales)
        steps[:i + 1] += 0.5001 * c.scales[1, 0]
    got = numbers(c.gpu.pool)[1]
    np.testing.assert_array_equal(got, c.pool[1])
    keys = got[0].reshape(heads, page, size) * c.scales[1, 0][:, None, None]
    off = np.abs(keys.transpose(1, 0, 2) - x)
    if kind == 'int8':
        assert (off <= steps[..., None]).all()
    else:  # at most 16 roundings
        assert (off <= 16 * (2.0**-4 * np.abs(x) * 1.01 + 2.0**-10 * c.scales[1, 0][None, :, None])).all()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('kind', ['int8', 'fp8'])
def test_append_of_what_is_not_finite_and_of_nothing(kind, dtype):
    rng = np.random.default_rng(4)
    c = Cache(rng, 4, 16, 2, 64, kind)
    k, _ = values(rng, (20, 2, 64), dtype)
    v = torch.zeros_like(k)
    k[3, 0, 5], k[4, 1, 6], k[5, 0, 7], v[6, 0, 0] = float('inf'), float('-inf'), float('nan'), float('nan')
    slots = np.arange(30, 50)
    with np.errstate(invalid='ignore'):
        O.append(c.pool, c.scales, k.float().numpy(), v.float().numpy(), slots, 16, kind, torch.finfo(TYPES[dtype]).max)
    c.gpu.append(k.cuda(), v.cuda(), gpu(slots))
    c.same()
    assert np.isfinite(c.scales).all()
    c.gpu.append(k[:0].cuda(), v[:0].cuda(), gpu([]))
    c.gpu.append(k.cuda(), v.cuda(), gpu(np.where(np.arange(20) % 2, -1, 64 + np.arange(20))))  # behind the pool's end: passed over
    c.same()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(rng, kind, dtype, page, size, kv, group, spans, window=0, scale=None, spare_rows=0, max_new=None, max_kv=None, bad=(), loud=1.0):
    """spans: [(cached tokens, rows)]"""
    pages = [-(-length // page) for length, _ in spans]
    blocks, wide = sum(pages) + 2, max(max(pages), 1)
    c = Cache(rng, blocks, page, kv, size, kind, garbage=True)
    ids, at = rng.permutation(blocks), 0
    table = np.full((len(spans), wide + 1), 10**9, np.int32)
    pool = c.gpu.pool.view(torch.uint8)
    for b, (length, _) in enumerate(spans):
        table[b, :pages[b]] = ids[at:at + pages[b]]
        at += pages[b]
        if kind == 'fp8':  # NaN patterns stay behind the last token alone
            for j in range(pages[b]):
                held = min(page, length - j * page)
                for which in (0, 1):
                    x = pool[int(table[b, j]), which].view(kv, *((page, size) if which == 0 else (size, page)))
                    x = x[:, :held] if which == 0 else x[:, :, :held]
                    x[(x & 0x7f) == 0x7f] = 0x38
    for b, j in bad:
        table[b, j] = [-1, blocks, 2**31 - 1][j % 3]
    c.pool = np.nan_to_num(numbers(c.gpu.pool), nan=0.0)
    cu = np.concatenate([[0], np.cumsum([n for _, n in spans])])
    lens = np.array([length for length, _ in spans])
    rows = int(cu[-1]) + spare_rows
    q = torch.from_numpy(rng.standard_normal((rows, kv * group, size)).astype(np.float32) * loud).to(TYPES[dtype])
    wide_q = torch.zeros((rows, kv * group + 3, size), dtype=TYPES[dtype], device='cuda')
    wide_q[:, :kv * group] = q.cuda()
    out = torch.full((rows, kv * group, size), 77.0, dtype=TYPES[dtype], device='cuda')
    t = torch.full((len(spans), wide + 5), -3, dtype=torch.int32, device='cuda')
    t[:, :wide + 1] = gpu(table)
    got = c.gpu.attention(wide_q[:, :kv * group], t[:, :wide], gpu(cu), gpu(lens), max_new or max(max(n for _, n in spans), 1), max_kv, window, scale, out)
    scale = size**-0.5 if scale is None else scale
    want, spread, worst = O.attention(q.float().numpy(), c.pool, c.scales, table[:, :wide], cu, lens, page, scale, window)
    got = numbers(got)
    assert (got[int(cu[-1]):] == 77).all()
    got, want, spread, worst = (x[:int(cu[-1])] for x in (got, want, spread, worst))
    # A score is a sum of `size` exact products in fp32 times a factor: off by size + 4 roundings of its terms (and a bfloat16 query's parts below
    # 2^-24 of its largest), a weight by twice that (itself and the sum) and some roundings; then 2^-11 as the weight becomes fp16, 2^-20 for
    # the sums over keys and parts, and one rounding of the result.
    z = (size + 4) * 2.0**-24 * worst + (2.0**-24 * size * worst if dtype == 'bf16' else 0)
    bound = (2 * z + 2.0**-11 + 2.0**-19) * spread * 1.01 + HALF[dtype] * np.abs(want) * 1.01 + 1e-7
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    return got


ONE = [(1, 1), (0, 0), (17, 1), (63, 1), (64, 1), (65, 1), (700, 1)]
FEW = [(3, 3), (40, 5), (0, 0), (129, 2), (70, 0), (1, 1)]
LONG = [(70, 70), (300, 33), (129, 1), (0, 0), (517, 130)]


@pytest.mark.parametrize('kind,dtype', [('int8', 'fp16'), ('fp8', 'bf16'), ('int8', 'bf16'), ('fp8', 'fp16')])
@pytest.mark.parametrize('spans', [ONE, FEW, LONG], ids=['one', 'few', 'long'])
@pytest.mark.parametrize('page,size,kv,group', [(64, 128, 2, 1), (16, 64, 1, 4), (32, 128, 2, 7), (128, 256, 1, 3), (64, 64, 1, 16), (16, 128, 1, 20)])
def test_attention(page, size, kv, group, spans, kind, dtype):
    check_attention(np.random.default_rng(page + size + group), kind, dtype, page, size, kv, group, spans, spare_rows=2)


@pytest.mark.parametrize('kind', ['int8', 'fp8'])
@pytest.mark.parametrize('spans', [ONE, FEW, LONG], ids=['one', 'few', 'long'])
@pytest.mark.parametrize('window', [1, 16, 63, 64, 65, 200, 100000])
def test_attention_window(window, spans, kind):
    check_attention(np.random.default_rng(window), kind, 'fp16', 32, 64, 2, 2, spans, window=window)


@pytest.mark.parametrize('kind,dtype,size', [('int8', 'fp16', 128), ('fp8', 'bf16', 64), ('int8', 'bf16', 256)])
@pytest.mark.parametrize('spans,max_kv', [([(9000, 1)], None), ([(9000, 1), (30, 1), (0, 0), (4097, 1)], 9000), ([(5000, 2), (1200, 1)], 70000), ([(2500, 1)], 0)])
def test_attention_split_over_workgroups(spans, max_kv, kind, dtype, size):
    check_attention(np.random.default_rng(size), kind, dtype, 64, size, 1, 3, spans, max_kv=max_kv, spare_rows=1)


@pytest.mark.parametrize('kind,dtype,size', [('int8', 'fp16', 128), ('fp8', 'bf16', 64), ('int8', 'bf16', 64), ('fp8', 'fp16', 128), ('int8', 'fp16', 256)])
@pytest.mark.parametrize('spans,max_kv,window', [([(500, 1)], None, 0), ([(290, 1), (0, 0), (511, 1), (64, 2)], None, 0), ([(900, 1), (1, 1)], None, 0), ([(3000, 1), (10, 1)], 400, 0),
                                                 ([(3000, 3), (449, 1)], None, 300)])
def test_attention_of_few_keys(spans, max_kv, window, kind, dtype, size):
    check_attention(np.random.default_rng(size), kind, dtype, 64, size, 2, 3, spans, max_kv=max_kv, window=window, spare_rows=1)


@pytest.mark.parametrize('size', [64, 256])
def test_attention_of_many_workgroups(size):
    """More than 32 row tiles an XCD, in numbers that do not divide it: every row is computed, and once."""
    spans = [(290, 270), (400, 300), (130, 130)] if size == 64 else [(140, 140), (200, 180)]
    check_attention(np.random.default_rng(size), 'int8', 'fp16', 64, size, 32 if size == 64 else 64, 1, spans)


@pytest.mark.parametrize('kind,dtype,size', [('int8', 'fp16', 128), ('fp8', 'bf16', 64), ('int8', 'bf16', 256)])
@pytest.mark.parametrize('window', [0, 1500])
def test_attention_prompts_split_over_workgroups(window, kind, dtype, size):
    """Few row tiles over long contexts, beside a single token, an empty request and one that sees little."""
    check_attention(np.random.default_rng(size), kind, dtype, 64, size, 1, 2, [(5000, 40), (3100, 1), (0, 0), (70, 30), (9, 20)], window=window, max_kv=9000, spare_rows=1)


@pytest.mark.parametrize('kind,dtype,size', [('int8', 'fp16', 128), ('fp8', 'bf16', 64), ('int8', 'bf16', 256)])
@pytest.mark.parametrize('kv,group', [(2, 1), (1, 4), (1, 20)])
@pytest.mark.parametrize('window', [0, 2200])
@pytest.mark.parametrize('spans', [[(4200, 1), (0, 100), (2500, 3), (70, 1), (0, 0), (2100, 40)], [(4200, 1), (3100, 30)]], ids=['many', 'two'])
def test_attention_of_tokens_beside_prompts(spans, window, kv, group, kind, dtype, size):
    check_attention(np.random.default_rng(len(spans) + window), kind, dtype, 64, size, kv, group, spans, window=window, spare_rows=3)


def test_attention_rows_that_see_nothing():
    """More rows than cached tokens: the first ones stand before the cache's beginning.  Lengths below zero and beyond the table."""
    rng = np.random.default_rng(8)
    for spans, window in (([(3, 5), (0, 4), (70, 90)], 0), ([(0, 1), (1, 2)], 0), ([(2, 40), (-5, 3)], 0), ([(3, 50), (1, 3)], 2**31 - 1), ([(3, 50), (1, 3)], 2)):
        got = check_attention(rng, 'int8', 'fp16', 16, 64, 1, 2, spans, window=window)
        assert (got[:max(spans[0][1] - spans[0][0], 0)] == 0).all()


def test_attention_passes_over_entries_that_are_no_blocks():
    rng = np.random.default_rng(9)
    for spans, bad in (([(200, 1), (64, 1)], [(0, 1), (0, 2), (1, 0)]), ([(200, 90), (10, 1)], [(0, 0), (0, 2)])):
        check_attention(rng, 'fp8', 'fp16', 32, 64, 2, 2, spans, bad=bad)


@pytest.mark.parametrize('size', [64, 128, 256])
@pytest.mark.parametrize('spans', [[(9, 3), (300, 2)], [(400, 2), (5000, 1)], [(100, 90), (700, 200), (40, 1)]], ids=['few', 'split', 'prompts'])
def test_attention_keeps_what_is_not_finite_to_its_row(spans, size):
    torch.manual_seed(size)
    pages = [-(-length // 64) for length, _ in spans]
    cache = P.PagedKV8Cache(torch.randint(-127, 128, (sum(pages), 2, 2, 64 * size), dtype=torch.int8, device='cuda'), torch.full((sum(pages), 2, 2), 1 / 127, device='cuda'), 64, size)
    table, ids = torch.zeros((len(spans), max(pages)), dtype=torch.int32, device='cuda'), torch.randperm(sum(pages), dtype=torch.int32, device='cuda')
    for b, n in enumerate(pages):
        table[b, :n] = ids[sum(pages[:b]):sum(pages[:b + 1])]
    rows = [new for _, new in spans]
    args = table, gpu(np.cumsum([0] + rows)), gpu([length for length, _ in spans]), max(rows)
    q = torch.randn((sum(rows), 4, size), device='cuda').half()
    clean, bad = cache.attention(q, *args), q.clone()
    bad[1, 2, 5], bad[-1, 0, 0] = float('nan'), float('nan')
    got = cache.attention(bad, *args)
    odd = torch.zeros(q.shape[:2], dtype=torch.bool, device='cuda')
    odd[1, 2] = odd[-1, 0] = True
    assert got[odd].isnan().all()
    # values are at most 1: each of the two is off by the weights' rounding, 2^-11, sums, 2^-19, and its own, 2^-11
    assert ((got[~odd].float() - clean[~odd].float()).abs() <= 2 * (2.0**-10 + 2.0**-19)).all()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_attention_of_far_scales(dtype):
    """Pages whose value scales are far from each other, and scores far beyond exp's range on both sides."""
    rng = np.random.default_rng(10)
    page, size, length = 16, 64, 200
    c = Cache(rng, 13, page, 1, size, 'int8')
    c.gpu.scales[:, 1, 0] = gpu(10.0**rng.uniform(-5, 1, 13), torch.float32)
    c.gpu.scales[:, 0, 0] = gpu(10.0**rng.uniform(-3, 0, 13), torch.float32)
    c.scales = c.gpu.scales.cpu().numpy()
    q = torch.from_numpy(rng.standard_normal((4, 2, size)).astype(np.float32)).to(TYPES[dtype])
    table, cu, lens = np.arange(13)[None], [0, 4], [length]
    got = numbers(c.gpu.attention(q.cuda(), gpu(table), gpu(cu), gpu(lens), 4))
    want, spread, worst = O.attention(q.float().numpy(), c.pool, c.scales, table, cu, lens, page, size**-0.5)
    bound = (2 * (2 * size + 4) * 2.0**-24 * worst + 2.0**-11 + 2.0**-19) * spread * 1.01 + HALF[dtype] * np.abs(want) * 1.01 + 1e-7
    assert (np.abs(got - want) <= bound).all()


def test_attention_queries_of_any_size_in_bfloat16():
    """Rows far beyond fp16's range on both sides, and rows of zeros; the softmax scale brings the scores back."""
    rng = np.random.default_rng(11)
    for loud, scale in ((1e20, 1e-21), (1e-20, 1e19), (0.0, None)):
        check_attention(rng, 'int8', 'bf16', 64, 128, 1, 2, [(90, 3), (1, 1)], scale=scale, loud=loud)


def test_attention_shares_follow_max_new():
    """Rows behind max_new are not computed and stay as they were."""
    rng = np.random.default_rng(12)
    c = Cache(rng, 4, 64, 1, 64, 'int8')
    q = torch.randn(40, 2, 64, device='cuda').half()
    args = (gpu([[0, 1], [2, 3]]), gpu([0, 30, 40]), gpu([100, 80]))
    whole = c.gpu.attention(q, *args, max_new=30)
    out = torch.full_like(q, 5.0)
    c.gpu.attention(q, *args, max_new=12, out=out)
    # the same rows in other tiles: both within the bound of each other's rounding
    assert torch.allclose(out[:12].float(), whole[:12].float(), rtol=2.0**-9, atol=2.0**-10) and (out[12:30] == 5).all()
    assert torch.allclose(out[30:].float(), whole[30:].float(), rtol=2.0**-9, atol=2.0**-10)


# ------------------------------------------------------------------------------------------------ 4-bit products
def check_product(rng, rows, n, k, group, dtype, strided=False):
    q = rng.integers(-8, 8, (n, k)).astype(np.int8)
    s = torch.from_numpy(rng.uniform(0.01, 0.2, (n, -(-k // group))).astype(np.float32)).to(TYPES[dtype])
    x = torch.from_numpy(rng.standard_normal((rows, k)).astype(np.float32)).to(TYPES[dtype])
    f = G.GroupQuantMatmul(torch.from_numpy(q).cuda(), s.cuda(), group)
    xg = x.cuda()
    if strided:
        wide = torch.full((rows, k + 24), float('nan'), dtype=TYPES[dtype], device='cuda')
        wide[:, :k] = xg
        y = torch.full((rows, n + 5), 9.0, dtype=TYPES[dtype], device='cuda')
        f(wide[:, :k], out=y[:, :n])
        assert (y[:, n:] == 9).all()
        y = y[:, :n]
    else:
        y = f(xg)
    want, terms, plain = O.group_product(x.float().numpy(), q, s.float().numpy(), group)
    # exact products summed in fp32: a rounding of the running sum for each step of 32 k and 32 for what is joined in a step and between waves;
    # bfloat16 sums 128 + u and takes 136 off within a group: at most 32 roundings of terms up to 280 |x| s
    bound = (k / 32 + 32) * 2.0**-24 * terms + HALF[dtype] * np.abs(want) * 1.01 + 1e-7
    if dtype == 'bf16':
        bound += 32 * 2.0**-24 * 280 * plain
    assert (np.abs(numbers(y) - want) <= bound).all(), float((np.abs(numbers(y) - want) / bound).max())


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('rows,n,k', [(1, 16, 32), (1, 1, 128), (1, 4096, 4096), (3, 100, 160), (16, 257, 992), (17, 64, 1024), (32, 130, 96), (33, 513, 2080), (64, 96, 11008),
                                      (65, 200, 256), (130, 300, 640), (257, 1000, 1312), (700, 31, 224), (1, 4097, 4128), (5, 2050, 1056), (1 << 19, 5, 32)])
def test_group_matmul(rows, n, k, group, dtype):
    check_product(np.random.default_rng(rows + n + k), rows, n, k, group, dtype)


@pytest.mark.parametrize('group,dtype', [(128, 'fp16'), (32, 'bf16'), (64, 'fp16')])
@pytest.mark.parametrize('rows,n', [(1, 1), (1, 4116), (1, 8195), (1, 12295), (1027, 1), (5, 4111), (5, 8207), (5, 12291), (1064, 17), (9, 4099), (17, 4118), (17, 6155), (1362, 65), (1381, 129), (17, 8196), (33, 6146), (1671, 130), (1633, 258), (33, 8197), (65, 6149), (129, 10943), (385, 12378), (2054, 17), (33, 10883), (33, 12338), (259, 10913)])
def test_group_matmul_in_every_form(rows, n, group, dtype):
    """Sizes at which each of the kernels' shapes is the quickest, k ending inside a tile."""
    check_product(np.random.default_rng(n), rows, n, 288, group, dtype)


@pytest.mark.parametrize('group,dtype', [(128, 'fp16'), (32, 'bf16'), (64, 'fp16')])
@pytest.mark.parametrize('k', [32, 128, 160, 256, 384, 512])
@pytest.mark.parametrize('rows,n', [(1500, 1100), (400, 1530), (2300, 2500)])
def test_group_matmul_of_few_k_tiles(rows, n, k, group, dtype):
    check_product(np.random.default_rng(rows + k), rows, n, k, group, dtype)


@pytest.mark.parametrize('rows,n', [(3, 40), (40, 100), (200, 300), (1500, 1100)])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_group_matmul_keeps_what_is_not_finite_to_its_row(rows, n, dtype):
    rng = np.random.default_rng(rows)
    q = torch.from_numpy(rng.integers(1, 8, (n, 160)).astype(np.int8)).cuda()
    f = G.GroupQuantMatmul(q, torch.from_numpy(rng.uniform(0.01, 0.2, (n, 3))).to(TYPES[dtype]).cuda(), 64)
    x = torch.from_numpy(rng.standard_normal((rows, 160)).astype(np.float32)).to(TYPES[dtype]).cuda()
    clean = f(x)
    bad = x.clone()
    bad[1, 33], bad[rows // 2, 150], bad[rows - 1, 0] = float('inf'), float('nan'), float('-inf')
    got, odd = f(bad), sorted({1, rows // 2, rows - 1})
    assert not got[odd].float().isfinite().any()
    if dtype == 'fp16' and rows > 3:
        assert (got[1] == float('inf')).all() and (got[rows - 1] == float('-inf')).all()
    same = [i for i in range(rows) if i not in odd]
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize('rows', [1, 9, 40, 300])
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
def test_group_matmul_strided(rows, dtype):
    check_product(np.random.default_rng(rows), rows, 203, 416, 64, dtype, strided=True)


def test_group_matmul_shapes_and_weights():
    rng = np.random.default_rng(1)
    w = torch.from_numpy(rng.standard_normal((70, 352)).astype(np.float32))
    w[3, 64:128] = 0
    q, s = G.quantize(w, 64)
    assert int(q.min()) >= -7 and int(q.max()) == 7 and float(s[3, 1]) == 1
    held = q.float() * s.float().repeat_interleave(64, 1)[:, :352]
    # half a step, and the scale's own rounding times 7
    assert bool(((held - w).abs() <= (0.5 + 7 * 2.0**-11) * s.float().repeat_interleave(64, 1)[:, :352] + 1e-6).all())
    f = G.GroupQuantMatmul.from_float(w.cuda(), 64)
    x = torch.randn(2, 3, 352, device='cuda').half()
    y = f(x)
    assert y.shape == (2, 3, 70) and torch.equal(y.view(6, 70), f(x.view(6, 352)))
    assert f(x[:, :0]).shape == (2, 0, 70)


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """A layer's attention as these operators make it: packed projection, pages, append, attention, projection back."""

    def __init__(self, rng, heads, kv, size, page, kind, dtype, blocks, seqs, wide):
        width = 256
        make = lambda n, k: G.GroupQuantMatmul.from_float(torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) / np.sqrt(k)).cuda(), 64, TYPES[dtype])
        self.qkv, self.o, self.heads, self.kv, self.size, self.width = make((heads + 2 * kv) * size, width), make(width, heads * size), heads, kv, size, width
        self.pool = P.DeviceBlockPool(blocks, page, seqs, wide)
        self.cache = P.PagedKV8Cache.empty(blocks, page, kv, size, CACHE[kind])
        self.rope = P.rope_table(wide * page, size)

    def step(self, x, new_lens, max_new, out=None):
        plan = self.pool.plan(new_lens, x.shape[0], out)
        qkv = self.qkv(x).view(-1, self.heads + 2 * self.kv, self.size)
        q, k, v = qkv[:, :self.heads], qkv[:, self.heads:self.heads + self.kv], qkv[:, self.heads + self.kv:]
        q = self.cache.append(k, v, plan.slot_map, plan.positions, self.rope, q, q_out=q)
        a = torch.zeros((x.shape[0], self.heads, self.size), dtype=x.dtype, device='cuda')
        self.cache.attention(q, self.pool.block_table, plan.cu_tokens, plan.lens, max_new, out=a)
        return self.o(a.view(-1, self.heads * self.size)), plan


@pytest.mark.parametrize('kind,dtype', [('int8', 'fp16'), ('fp8', 'bf16')])
def test_steps_of_a_layer_against_64_bits(kind, dtype):
    """Prompts in portions, tokens, requests that end and come: every step's result against float64 over the whole history, which knows no cache.  The
    cache's 8 bits are most of the difference: its values are off by their rounding (int8: half of 1/127 of a page's largest, e4m3: 2^-4), keys
    move the softmax by as much times the queries' size.  With unit inputs that leaves a tenth (a fifth) of the result's root mean square."""
    rng = np.random.default_rng(21)
    layer = Layer(rng, 4, 2, 64, 16, kind, dtype, 60, 3, 20)
    dense = lambda f: f(torch.eye(f.k, device='cuda').to(f.dtype)).double().cpu().numpy()  # the weights as they are, rounded once
    wq, wo = dense(layer.qkv), dense(layer.o)
    rope = layer.rope.double().cpu().numpy()
    hist = [np.zeros((0, 256)) for _ in range(3)]
    for new in ([37, 5, 0], [20, 1, 18], [1, 1, 1], [1, -1, 1], [1, 33, 1], [1, 1, 1], [40, 0, 1]):
        n = sum(max(v, 0) for v in new)
        x = torch.from_numpy(rng.standard_normal((n + 2, 256)).astype(np.float32)).to(TYPES[dtype]).cuda()
        y, plan = layer.step(x, gpu(new), 40)
        assert int(plan.status) == 0
        row = 0
        for b, add in enumerate(new):
            if add < 0:
                hist[b] = np.zeros((0, 256))
                continue
            hist[b] = np.concatenate([hist[b], x[row:row + add].double().cpu().numpy()])
            if add == 0:
                continue
            z = (hist[b] @ wq).reshape(-1, 8, 64)
            t = len(z)
            z[:, :6] = O.rotate(z[:, :6], rope[:t], False)
            want = np.zeros((add, 4, 64))
            for h in range(4):
                s = z[t - add:, h] @ z[:, 4 + h // 2].T / 8
                s[np.arange(t)[None] > np.arange(t - add, t)[:, None]] = -np.inf
                p = np.exp(s - s.max(-1, keepdims=True))
                want[:, h] = p / p.sum(-1, keepdims=True) @ z[:, 6 + h // 2]
            want = want.reshape(add, 256) @ wo
            got = y[row:row + add].double().cpu().numpy()
            off = np.sqrt(np.mean((got - want)**2) / np.mean(want**2))
            assert off < (0.1 if kind == 'int8' else 0.2), (new, b, off)
            row += add


def test_steps_captured_and_replayed():
    """A decoding step as a graph: lengths and free list live on the GPU, so the same graph is every next step.  Bits as of eager steps, with eager work
    and synchronisation between the replays."""
    outs = []
    for captured in (False, True):
        rng = np.random.default_rng(33)
        layer = Layer(rng, 4, 2, 64, 16, 'int8', 'fp16', 60, 3, 20)
        layer.step(torch.from_numpy(rng.standard_normal((60, 256)).astype(np.float32)).half().cuda(), gpu([40, 15, 3]), 40)
        x, new = torch.zeros((3, 256), dtype=torch.float16, device='cuda'), gpu([1, 1, 1])
        plan = P.StepPlan(3, 3, 'cuda', lens=layer.pool.lens, ring_state=layer.pool.ring_state)
        feed = [torch.from_numpy(rng.standard_normal((3, 256)).astype(np.float32)).half().cuda() for _ in range(20)]
        if captured:
            g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
                y, _ = layer.step(x, new, 1, plan)
            torch.cuda.synchronize()
        got = []
        for i, f in enumerate(feed):
            x.copy_(f)
            if captured:
                g.replay()
            else:
                y, _ = layer.step(x, new, 1, plan)
            got.append(y.clone())
            torch.randn(1000, device='cuda').sum()
            if i % 3 == 0:
                torch.cuda.synchronize()
        assert int(plan.status) == 0 and layer.pool.lens.tolist() == [60, 35, 23]
        outs.append(torch.stack(got).cpu())
    assert torch.equal(outs[0], outs[1])


def test_two_streams_at_once():
    """Two layers' steps side by side on streams of their own give what each gives alone."""
    def make(seed):
        rng = np.random.default_rng(seed)
        return Layer(rng, 4, 1, 128, 32, 'fp8', 'fp16', 200, 2, 90), torch.from_numpy(rng.standard_normal((2300, 256)).astype(np.float32)).half().cuda()

    def steps(layer, x):
        a, _ = layer.step(x, gpu([1500, 800]), 1500)
        return [a] + [layer.step(x[i:i + 2], gpu([1, 1]), 1)[0] for i in range(6)]

    alone = [steps(*make(s)) for s in (1, 2)]
    pair, streams = [make(s) for s in (1, 2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    both = []
    for (layer, x), s in zip(pair, streams):
        with torch.cuda.stream(s):
            both.append(steps(layer, x))
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('spans', [[(0, 5), (70, 1), (300, 2)], [(100, 300), (9, 1)], [(9000, 1)], [(9000, 100)]], ids=['few', 'prompt', 'split', 'split prompt'])
def test_attention_in_place_of_its_queries(spans, dtype):
    """out is q, both a view into a packed projection: the bits are those of the call with a result of its own."""
    torch.manual_seed(5)
    pages = [-(-(past + new) // 64) for past, new in spans]
    cache = P.PagedKV8Cache(torch.randint(-127, 128, (sum(pages), 2, 2, 64 * 128), dtype=torch.int8, device='cuda'), torch.rand((sum(pages), 2, 2), device='cuda') * 1e-2, 64, 128)
    table = torch.zeros((len(spans), max(pages)), dtype=torch.int32, device='cuda')
    ids = torch.randperm(sum(pages), dtype=torch.int32, device='cuda')
    for b, n in enumerate(pages):
        table[b, :n] = ids[sum(pages[:b]):sum(pages[:b + 1])]
    rows = [new for _, new in spans]
    qkv = torch.randn((sum(rows), 8, 128), device='cuda').to(TYPES[dtype])
    q, kept = qkv[:, :6], qkv.clone()
    args = table, gpu(np.cumsum([0] + rows)), gpu([past + new for past, new in spans]), max(rows)
    want = cache.attention(q, *args)
    assert cache.attention(q, *args, out=q) is q
    assert torch.equal(q, want) and torch.equal(qkv[:, 6:], kept[:, 6:])


def test_copies_have_tensors_of_their_own():
    torch.manual_seed(3)
    mm, cache = G.GroupQuantMatmul.from_float(torch.randn((50, 96), device='cuda'), 32), P.PagedKV8Cache.empty(2, 16, 1, 64)
    x, kv, q = torch.randn((3, 96), device='cuda').half(), torch.randn((5, 2, 64), device='cuda').half(), torch.randn((5, 2, 64), device='cuda').half()
    table, cu, lens = gpu([[1]]), gpu([0, 5]), gpu([5])
    cache.append(kv[:, :1], kv[:, 1:], gpu(range(16, 21)))
    want, seen = mm(x), cache.attention(q, table, cu, lens, 5)
    for make in (copy.copy, copy.deepcopy, lambda thing: pickle.loads(pickle.dumps(thing))):
        mm2, cache2 = make(mm), make(cache)
        if make is not copy.copy:
            assert mm2.packed.data_ptr() != mm.packed.data_ptr() and cache2.pool.data_ptr() != cache.pool.data_ptr()
            kept = [t.clone() for t in (mm.packed, mm.scales, cache.pool, cache.scales)]
            for t in (mm.packed, mm.scales, cache.pool, cache.scales):
                t.zero_()
        assert torch.equal(mm2(x), want) and torch.equal(cache2.attention(q, table, cu, lens, 5), seen)
        if make is not copy.copy:
            for t, was in zip((mm.packed, mm.scales, cache.pool, cache.scales), kept):
                t.copy_(was)


def test_tensors_of_the_objects_stay():
    cache, mm, plan = P.PagedKV8Cache.empty(2, 16, 1, 64), G.GroupQuantMatmul(torch.zeros((1, 32), dtype=torch.int8, device='cuda'), torch.ones((1, 1), device='cuda').half(), 32), P.StepPlan(1, 1)
    for thing, name in ((cache, 'pool'), (cache, 'scales'), (mm, 'scales'), (mm, 'packed'), (plan, 'lens'), (plan, 'slot_map')):
        with pytest.raises(AttributeError, match='stays'):
            setattr(thing, name, getattr(thing, name).clone())


def test_wrappers_refuse():
    c = P.PagedKV8Cache.empty(4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device='cuda')
    s, rope = gpu([0, 1, 2]), P.rope_table(8, 64)
    with pytest.raises(TypeError):
        c.append(k.float(), k.float(), s)
    for bad in ((k[:, :1], k, s), (k, k[..., :32], s), (k, k.transpose(1, 2).contiguous().transpose(1, 2), s), (k, k, s.long()), (k, k, s[:2]), (k.cpu(), k, s), (k, k.bfloat16(), s)):
        with pytest.raises(ValueError):
            c.append(*bad)
    with pytest.raises(ValueError):
        c.append(k, k, s, q=k)
    with pytest.raises(ValueError):
        c.append(k, k, s, rope=rope)
    with pytest.raises(RuntimeError, match='aligned'):
        c.append(torch.zeros(3 * 128 + 1, dtype=torch.float16, device='cuda')[1:].view(3, 2, 64), k, s)
    with pytest.raises(RuntimeError, match='rot_dim'):
        c.append(k, k, s, s, P.rope_table(8, 40), k)
    t, cu, n = gpu([[0, 1]]), gpu([0, 3]), gpu([3])
    with pytest.raises(RuntimeError, match='kv_heads'):
        c.attention(torch.zeros(3, 3, 64, dtype=torch.float16, device='cuda'), t, cu, n, 3)
    with pytest.raises(RuntimeError, match='max_new'):
        c.attention(k, t, cu, n, 0)
    for bad in ((k, t.long(), cu, n), (k, t[:, ::2], cu[:1], n), (k[..., :32], t, cu, n), (k, t, cu, n.float()), (k, gpu([[0, 1], [2, 3]]).t(), cu, n)):
        with pytest.raises(ValueError):
            c.attention(*bad, max_new=3)
    for bad in (dict(page_size=48), dict(head_size=96), dict(pool=c.pool.float()), dict(scales=c.scales[:2])):
        with pytest.raises(ValueError):
            P.PagedKV8Cache(**{**dict(pool=c.pool, scales=c.scales, page_size=16, head_size=64), **bad})
    pool = P.DeviceBlockPool(4, 16, 2, 3)
    out = P.StepPlan(2, 5)
    for bad in ((gpu([1, 1]).long(), 5, out), (gpu([1]), 5, out), (gpu([1, 1]), 4, out), (gpu([1, 1]).cpu(), 5, out)):
        with pytest.raises(ValueError):
            pool.plan(*bad)
    with pytest.raises(AttributeError):
        out.slot_map = gpu([1])
    with pytest.raises(RuntimeError, match='page_size'):
        P.plan_step(n, n, gpu([0, 1]), gpu([0, 2]), t, 24, 3)
    f = G.GroupQuantMatmul(torch.zeros(8, 64, dtype=torch.int8, device='cuda'), torch.ones(8, 1, dtype=torch.float16, device='cuda'), 64)
    x = torch.zeros(64, 64, dtype=torch.float16, device='cuda')
    for bad in (x[:, :32], x.float(), x.cpu(), x.t()):
        with pytest.raises(ValueError):
            f(bad)
    with pytest.raises(ValueError):
        f(x, out=torch.zeros(64, 9, dtype=torch.float16, device='cuda'))
    with pytest.raises(ValueError):
        G.pack(torch.full((4, 64), 8, dtype=torch.int8), torch.ones(4, 1).half(), 64)
    with pytest.raises(RuntimeError, match='aligned'):
        f(torch.zeros(2 * 64 + 1, dtype=torch.float16, device='cuda')[1:].view(2, 64))
