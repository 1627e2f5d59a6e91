"""The operators of a quantised serving step, as cases that a timing program can prepare, run and check.

A step of a server that keeps many requests in little memory: the pages that the step's tokens go to are taken from a free list on the
GPU (`plan`), the step's keys and values enter a paged cache held in 8 bits with a scale for each page and head (`append`), the
queries attend to that cache (`attention`), and the linear layers around it have 4-bit weights with a scale for each group of a row
(`product`).

A plan case is {op, seqs, new, past, page, decode, release, salt}: `seqs` requests with up to `past` tokens held, of which a share `release`
ends in this step, a share `decode` brings one token and the others a portion of their prompt of up to `new` tokens.
An append or attention case is {op, seqs, new, past, page, heads, kv_heads, dim, dtype, cache, salt} and `rot` (rotated dimensions) or
`window` (0: none) and `decode`.  A product case is {op, rows, n, k, group, dtype}.
`salt` draws the lengths, the seed of a pass draws all values."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.realpath(__file__)))
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}
LARGEST = {'int8': 127.0, 'fp8': 448.0}  # the largest value that a stored element stands for, in units of its scale
FLOOR = 2.0**-100  # a page's largest magnitude counts as at least this: scales are never zero


# ------------------------------------------------------------------------------------------------------------------ the cases
def _plan(name, seqs, new, past, page, decode, release, salt=1):
    return dict(name=name, op='plan', seqs=seqs, new=new, past=past, page=page, decode=decode, release=release, salt=salt)


def _append(name, seqs, new, past, page, heads, kv_heads, dim, dtype, cache, rot, decode=0.0, salt=1):
    return dict(name=name, op='append', seqs=seqs, new=new, past=past, page=page, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                cache=cache, rot=rot, decode=decode, salt=salt)


def _attention(name, seqs, new, past, page, heads, kv_heads, dim, dtype, cache, window=0, decode=0.0, salt=1):
    return dict(name=name, op='attention', seqs=seqs, new=new, past=past, page=page, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                cache=cache, window=window, decode=decode, salt=salt)


def _product(name, rows, n, k, group, dtype):
    return dict(name=name, op='product', rows=rows, n=n, k=k, group=group, dtype=dtype)


def listed():
    return [
        # sixteen users generate: one token each, now and then a new page; latency counts
        _plan('plan_tokens', 16, 1, 2000, 64, 1.0, 0.0),
        # a server changes over: many requests, half of them reading prompts, some ending
        _plan('plan_requests', 512, 300, 1500, 16, 0.5, 0.1),
        # a decoded token of each of 64 users, keys and values entering pages that hold some already
        _append('append_tokens', 64, 1, 62, 64, 32, 8, 128, 'fp16', 'int8', 128),
        # portions of long prompts, pages filled whole
        _append('append_prompts', 5, 1500, 700, 64, 32, 8, 128, 'bf16', 'fp8', 128),
        # LLaMA-7B answers one user behind a 1024-token context
        _attention('attention_chat', 1, 1, 1031, 64, 32, 32, 128, 'fp16', 'int8'),
        # 48 users generate over contexts of different lengths, grouped heads
        _attention('attention_batch', 48, 1, 8000, 32, 32, 8, 128, 'bf16', 'fp8'),
        # one token behind a very long document
        _attention('attention_long', 1, 1, 131071, 128, 32, 8, 128, 'fp16', 'int8'),
        # prompts of LLaMA-7B arrive in portions behind what is cached
        _attention('attention_prompts', 3, 1024, 2500, 64, 32, 32, 128, 'fp16', 'int8'),
        # LLaMA-7B's output projection for one token
        _product('product_token', 1, 4096, 4096, 128, 'fp16'),
        # its feed-forward's way back for eight tokens, with small groups
        _product('product_down', 8, 4096, 11008, 64, 'bf16'),
        # its queries, keys and values for a batch of 24 users
        _product('product_batch', 24, 12288, 4096, 128, 'fp16'),
        # its feed-forward over a prompt: the matrix product at its largest
        _product('product_prompt', 1024, 11008, 4096, 128, 'fp16'),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng: random.Random):
    """A case of the same ranges: any operator, from one token to the longest prompts and contexts, any of the head layouts and types."""
    op = rng.choice(['plan', 'append', 'attention', 'attention', 'product', 'product'])
    most = {}
    for m in ('bytes', 'flops'):
        most[m] = max(work(c)[m] for c in listed() if c['op'] == op)
    while True:
        salt = rng.randrange(1 << 30)
        dtype, page = rng.choice(['fp16', 'fp16', 'bf16']), rng.choice([16, 32, 64, 128])
        cache, dim = rng.choice(['int8', 'int8', 'fp8']), rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 32])
        heads = kv * (1 if kv == 32 else rng.choice([1, 2, 3, 4, 5, 8]))
        decode = rng.choice([0.0, 0.5, 1.0])
        if op == 'plan':
            c = _plan(None, _log_int(rng, 1, 1024), _log_int(rng, 1, 4096), _log_int(rng, 1, 8000), page, decode, rng.choice([0.0, 0.1, 0.5]), salt)
        elif op == 'append':
            rot = rng.choice([0, dim // 2, dim])
            c = _append(None, _log_int(rng, 1, 128), _log_int(rng, 1, 2000), _log_int(rng, 1, 1000), page, heads, kv, dim, dtype, cache, rot, decode, salt)
        elif op == 'attention':
            window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
            new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 2048)
            c = _attention(None, _log_int(rng, 1, 96), new, _log_int(rng, 1, 100000), page, heads, kv, dim, dtype, cache, window, decode, salt)
        else:
            group = rng.choice([32, 64, 128])
            rows = _log_int(rng, 1, 16) if rng.random() < 0.6 else _log_int(rng, 17, 1024)
            c = _product(None, rows, _log_int(rng, 64, 12288), 32 * _log_int(rng, 4, 344), group, dtype)
        del c['name']
        if held(c) <= 2 ** 30 and all(work(c)[m] <= most[m] for m in ('bytes', 'flops')):
            return c


def lengths(case):
    """Per request, the tokens that the cache holds before the step and those that the step brings (-1: the request ends)."""
    rng = random.Random(case['salt'])
    past, new = [], []
    for i in range(case['seqs']):
        past.append(rng.randint(case['past'] // 2, case['past']))
        if i and rng.random() < case.get('release', 0.0):
            new.append(-1)
        elif i and rng.random() < case['decode']:
            new.append(1)
        else:
            new.append(rng.randint((case['new'] + 1) // 2, case['new']) if i else case['new'])
    past[0] = case['past']
    return past, new


def _pages(tokens, page):
    return -(-tokens // page)


def held(case):
    """The elements that an append or attention case's cache has."""
    if case['op'] not in ('append', 'attention'):
        return 0
    past, new = lengths(case)
    return 2 * case['kv_heads'] * case['dim'] * case['page'] * sum(_pages(p + n, case['page']) for p, n in zip(past, new))


def _attended(case, past, new):
    """Keys that the queries of one request see, together, and keys that any of them sees."""
    w = case['window'] or past + new
    return sum(min(w, past + i + 1) for i in range(new)), min(past + new, w + new - 1)


def work(case):
    op = case['op']
    if op == 'product':
        m, n, k = case['rows'], case['n'], case['k']
        return {'bytes': 2 * m * (n + k) + n * k / 2 + 2 * n * _pages(k, case['group']), 'flops': 2 * m * n * k}
    past, new = lengths(case)
    tokens = sum(n for n in new if n > 0)
    if op == 'plan':  # lengths in, lengths and sums out, pages from the list into the table, a slot and a position for each token
        pages = sum(_pages(p, case['page']) if n < 0 else _pages(p + n, case['page']) - _pages(p, case['page']) for p, n in zip(past, new))
        return {'bytes': 16 * case['seqs'] + 8 * pages + 8 * tokens, 'flops': 0}
    h, kv, d = case['heads'], case['kv_heads'], case['dim']
    if op == 'append':
        return {'bytes': tokens * ((4 * h if case['rot'] else 0) + 4 * kv + 2 * kv) * d + tokens * 4 * (2 + case['rot']), 'flops': 8 * tokens * (h + 2 * kv) * d}
    seen = [_attended(case, p, n) for p, n in zip(past, new)]
    return {'bytes': 4 * tokens * h * d + 2 * kv * d * sum(s[1] for s in seen), 'flops': 4 * h * d * sum(s[0] for s in seen)}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = {'case': case}
    globals()['_prepare_' + case['op']](case, seed, g, s)
    if own:
        path = os.path.join(ROOT, 'trtllm-llama_amd')
        if path not in sys.path:
            sys.path.insert(0, path)
        globals()['_ready_' + case['op']](s)
    return s


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _tables(case, seed, past, new, spare):
    """Block ids of every request, in an order without meaning, behind each other in a shuffled pool; the ids that are left."""
    need = [_pages(p + max(n, 0), case['page']) for p, n in zip(past, new)]
    ids = np.random.default_rng(seed).permutation(sum(need) + spare).astype(np.int32)
    table, at = np.zeros((len(need), max(need)), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, ids


def _prepare_plan(case, seed, g, s):
    past, new = lengths(case)
    page = case['page']
    table, ids = _tables(case, seed, past, new, 7)
    have = [_pages(p, page) for p in past]
    blocks = len(ids)
    for i, h in enumerate(have):
        table[i, h:] = 0
    taken = {int(b) for i, h in enumerate(have) for b in table[i, :h]}
    free = [int(b) for b in ids if int(b) not in taken]  # what no request holds yet
    head = int(np.random.default_rng(seed + 1).integers(0, blocks))
    ring = np.zeros(blocks, np.int32)
    ring[(head + np.arange(len(free))) % blocks] = free
    tokens = sum(n for n in new if n > 0)
    s.update(lens=_ints(past), new=_ints(new), ring=_ints(ring), ring_state=_ints([head, len(free)]), table=_ints(table), tokens=tokens + 3)


def _packed(case, tokens, g):
    """Rows of queries, keys and values side by side, as a projection leaves them: a few channels are much larger than the others."""
    h, kv, d = case['heads'], case['kv_heads'], case['dim']
    x = torch.randn((tokens, h + 2 * kv, d), generator=g, device='cuda')
    x *= 0.5 + 4 * (torch.rand((1, h + 2 * kv, d), generator=g, device='cuda') > 0.97)
    return x.to(TYPES[case['dtype']])


def _quantised(x, cache):
    """Values in 8 bits under one scale for each [block, key or value, head]: x [blocks, 2, kv_heads, page * dim]."""
    scale = x.abs().amax(-1).clamp_min(FLOOR) / LARGEST[cache]
    x = x / scale[..., None]
    return (x.round().to(torch.int8) if cache == 'int8' else x.to(torch.float8_e4m3fn)), scale


def _pool(case, blocks, g):
    """A pool that is full of earlier tokens: keys of a head [page, dim], values [dim, page]."""
    kv, d, page = case['kv_heads'], case['dim'], case['page']
    elem = torch.int8 if case['cache'] == 'int8' else torch.float8_e4m3fn
    pool = torch.empty((blocks, 2, kv, page * d), dtype=elem, device='cuda')
    scales = torch.empty((blocks, 2, kv), dtype=torch.float32, device='cuda')
    step = max(1, (1 << 26) // (2 * kv * page * d))
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        x = torch.randn((n, 2, kv, page * d), generator=g, device='cuda')
        x *= torch.rand((n, 2, kv, 1), generator=g, device='cuda') + 0.5
        q, t = _quantised(x, case['cache'])
        pool[b:b + n], scales[b:b + n] = q, t
    return pool, scales


def _prepare_append(case, seed, g, s):
    past, new = lengths(case)
    page, rot = case['page'], case['rot']
    table, ids = _tables(case, seed, past, new, 1)
    slots, places = [], []
    for i, (p, n) in enumerate(zip(past, new)):
        at = np.arange(p, p + n)
        slots.append(table[i, at // page].astype(np.int64) * page + at % page)
        places.append(at)
    slots, places = np.concatenate(slots), np.concatenate(places)
    angle = np.arange(max(p + n for p, n in zip(past, new)))[:, None] * 10000.0**(-np.arange(rot // 2) * 2.0 / max(rot, 1))
    qkv = _packed(case, len(slots), g)
    h, kv = case['heads'], case['kv_heads']
    pool, scales = _pool(case, len(ids), g)
    s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], slots=_ints(slots), places=_ints(places), pool=pool, scales=scales,
             rope=torch.tensor(np.stack([np.cos(angle), np.sin(angle)], -1), dtype=torch.float32, device='cuda'))


def _prepare_attention(case, seed, g, s):
    past, new = lengths(case)
    table, ids = _tables(case, seed, past, new, 1)
    pool, scales = _pool(case, len(ids), g)
    q = torch.randn((sum(new), case['heads'], case['dim']), generator=g, device='cuda') * 1.5
    s.update(q=q.to(TYPES[case['dtype']]), pool=pool, scales=scales, table=_ints(table), cu=_ints(np.concatenate([[0], np.cumsum(new)])),
             lens=_ints([p + n for p, n in zip(past, new)]), past=past, new=new)


def _prepare_product(case, seed, g, s):
    m, n, k, group = case['rows'], case['n'], case['k'], case['group']
    t = TYPES[case['dtype']]
    w = torch.randint(-8, 8, (n, k), generator=g, device='cuda', dtype=torch.int8)
    scales = ((torch.rand((n, _pages(k, group)), generator=g, device='cuda') + 0.5) * (0.3 / math.sqrt(k))).to(t)
    s.update(x=torch.randn((m, k), generator=g, device='cuda').to(t), w=w, scales=scales)


# ------------------------------------------------------------------------------------------------------------------ the framework's kernels
def _ready_plan(s):
    from tensorrt_llm.runtime import paged_kv8
    s['out'] = paged_kv8.StepPlan(s['lens'].numel(), s['tokens'], 'cuda')


def _ready_append(s):
    from tensorrt_llm.runtime import paged_kv8
    c = s['case']
    s['cache'] = paged_kv8.PagedKV8Cache(s['pool'], s['scales'], c['page'], c['dim'])


def _ready_attention(s):
    _ready_append(s)


def _ready_product(s):
    from tensorrt_llm.quantization import group
    s['linear'] = group.GroupQuantMatmul(s.pop('w'), s['scales'], s['case']['group'])


def _own_plan(s):
    from tensorrt_llm.runtime import paged_kv8
    p = paged_kv8.plan_step(s['lens'], s['new'], s['ring'], s['ring_state'], s['table'], s['case']['page'], s['tokens'], out=s['out'])
    return {'lens': p.lens, 'cu': p.cu_tokens, 'slots': p.slot_map, 'places': p.positions, 'ring_state': p.ring_state, 'status': p.status,
            'table': s['table'], 'ring': s['ring']}


def _own_append(s):
    rot = s['case']['rot']
    q = s['cache'].append(s['k'], s['v'], s['slots'], **(dict(q=s['q'], positions=s['places'], rope=s['rope']) if rot else {}))
    return _told(s, q if rot else None)


def _own_attention(s):
    return s['cache'].attention(s['q'], s['table'], s['cu'], s['lens'], max_new=max(s['new']), max_kv=max(p + n for p, n in zip(s['past'], s['new'])),
                                window=s['case']['window'])


def _own_product(s):
    return s['linear'](s['x'])


# ------------------------------------------------------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    lens, new, ring, state, table, page, cap = s['lens'], s['new'], s['ring'], s['ring_state'], s['table'], s['case']['page'], s['tokens']
    wide, blocks = table.shape[1], ring.numel()
    gone, step = new < 0, new.clamp_min(0)
    have = (lens + (page - 1)) // page
    after = torch.where(gone, torch.zeros_like(lens), lens + step)
    need = torch.where(gone, have, (lens + step + (page - 1)) // page)
    takes, gives = need - have, torch.where(gone, have, torch.zeros_like(have))
    ends, took, gave = step.cumsum(0), takes.cumsum(0), gives.cumsum(0)
    status = (need.max() > wide).int() + 2 * (took[-1] > state[1]).int() + 4 * (ends[-1] > cap).int()
    good = status == 0
    col = torch.arange(wide, device='cuda')[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None]) & good
    at = (state[0] + (took - takes)[:, None] + col - have[:, None]) % blocks
    table.copy_(torch.where(fresh, ring[at], table))
    back = gone[:, None] & (col < have[:, None]) & good
    to = torch.where(back, (state[0] + state[1] + (gave - gives)[:, None] + col) % blocks, blocks)
    longer = torch.cat([ring, ring[:1]])
    longer[to.reshape(-1)] = table.reshape(-1)
    ring.copy_(longer[:blocks])
    t = torch.arange(cap, device='cuda')
    seq = torch.searchsorted(ends, t, right=True).clamp_max(len(lens) - 1)
    place = lens[seq] + t - (ends - step)[seq]
    live = (t < ends[-1]) & good
    slot = table[seq, (place // page).clamp(0, wide - 1)] * page + place % page
    return {'lens': torch.where(good, after, lens).int(), 'cu': torch.where(good, torch.cat([ends.new_zeros(1), ends]), 0).int(), 'slots': torch.where(live, slot, -1).int(),
            'places': torch.where(live, place, -1).int(),
            'ring_state': torch.where(good, torch.stack([(state[0] + took[-1]) % blocks, state[1] - took[-1] + gave[-1]]), state).int(),
            'status': status.int().reshape(1), 'table': table, 'ring': ring}


def _rotated(x, s):
    """The halves of the first `rot` dimensions turned against each other."""
    rot = s['case']['rot']
    x = x.float()
    if not rot:
        return x
    c, n = s['rope'][s['places'].long()].unbind(-1)
    c, n, a, b = c[:, None], n[:, None], x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * n, b * c + a * n, x[..., rot:]], -1)


def _told(s, q):
    """The queries as rotated, the scales, and the cache as the values that it stands for."""
    pool, scales = s['pool'], s['scales']
    held_ = pool if s['case']['cache'] == 'int8' else pool.to(torch.float16)
    values = torch.mul(held_, scales[..., None], out=torch.empty(pool.shape, dtype=torch.float16, device='cuda'))
    return [values, scales] + ([q] if q is not None else [])


def _plain_append(s):
    c = s['case']
    kv, d, page, top = c['kv_heads'], c['dim'], c['page'], LARGEST[c['cache']]
    pool, scales = s['pool'], s['scales']
    blocks = pool.shape[0]
    x = torch.stack([_rotated(s['k'], s), s['v'].float()], 1)  # [tokens, 2, kv_heads, dim]
    slots = s['slots'].long()
    block, off = slots // page, slots % page
    first = torch.full((blocks, ), page, device='cuda', dtype=torch.int64).scatter_reduce(0, block, off, 'amin')
    amax = torch.zeros((blocks, 2, kv), device='cuda').index_reduce(0, block, x.abs().amax(-1), 'amax')
    old = torch.where((first > 0)[:, None, None], scales, torch.zeros_like(scales))
    scale = torch.where((first < page)[:, None, None], torch.maximum(old, amax.clamp_min(FLOOR) / top), scales)
    ratio = torch.where((first < page)[:, None, None], old / scale, torch.ones_like(scale))
    was = pool.float()
    keys, values = was[:, 0].view(blocks, kv, page, d) * ratio[:, 0, :, None, None], was[:, 1].view(blocks, kv, d, page) * ratio[:, 1, :, None, None]
    behind = torch.arange(page, device='cuda')[None, :] >= first[:, None]  # [blocks, page]: not held before the step
    keys = torch.where(behind[:, None, :, None], was[:, 0].view(blocks, kv, page, d), keys)
    values = torch.where(behind[:, None, None, :], was[:, 1].view(blocks, kv, d, page), values)
    x = x / scale[block][..., None]
    keys[block, :, off], values[block, :, :, off] = x[:, 0], x[:, 1]
    both = torch.stack([keys.reshape(blocks, kv, -1), values.reshape(blocks, kv, -1)], 1)
    pool.copy_(both.round().to(torch.int8) if c['cache'] == 'int8' else both.to(torch.float8_e4m3fn))
    scales.copy_(scale)
    return _told(s, _rotated(s['q'], s).to(s['q'].dtype) if c['rot'] else None)


def _gathered(s, table):
    """Keys and values of whole tables: table [.., pages] -> 2 x [.., kv_heads, pages * page, dim] in 32 bits."""
    c = s['case']
    kv, d, page = c['kv_heads'], c['dim'], c['page']
    x = s['pool'][table.long()].float() * s['scales'][table.long()][..., None]  # [.., pages, 2, kv, page * dim]
    k = x[..., 0, :, :].unflatten(-1, (page, d)).transpose(-4, -3)
    v = x[..., 1, :, :].unflatten(-1, (d, page)).transpose(-2, -1).transpose(-4, -3)
    return k.flatten(-3, -2).contiguous(), v.flatten(-3, -2).contiguous()


def _softmax_rows(scores, seen):
    scores = scores.masked_fill(~seen, float('-inf'))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_attention(s):
    c = s['case']
    h, kv, d, window = c['heads'], c['kv_heads'], c['dim'], c['window']
    q = s['q'].float() / math.sqrt(d)
    if max(s['new']) == 1:  # a token each: all requests side by side, the shorter ones masked behind their ends
        q = q.view(-1, kv, h // kv, d)
        k, v = _gathered(s, s['table'])
        at = torch.arange(k.shape[2], device='cuda')[None, :]
        seen = (at < s['lens'][:, None]) & (at >= s['lens'][:, None] - (window or k.shape[2]))
        p = _softmax_rows(torch.matmul(q, k.transpose(-1, -2).contiguous()), seen[:, None, None])
        return torch.matmul(p, v).view(-1, h, d).to(s['q'].dtype)
    out, row = [], 0
    for i, (past, new) in enumerate(zip(s['past'], s['new'])):
        n = past + new
        k, v = _gathered(s, s['table'][i, :_pages(n, c['page'])])
        rows = q[row:row + new].view(new, kv, h // kv, d).transpose(0, 1).reshape(kv, new * (h // kv), d)
        at, place = torch.arange(n, device='cuda')[None, :], torch.arange(past, n, device='cuda').repeat_interleave(h // kv)[:, None]
        seen = (at <= place) & (at > place - (window or n))
        p = _softmax_rows(torch.matmul(rows, k[:, :n].transpose(-1, -2).contiguous()), seen[None])
        out.append(torch.matmul(p, v[:, :n]).view(kv, new, h // kv, d).transpose(0, 1).reshape(new, h, d))
        row += new
    return torch.cat(out).to(s['q'].dtype)


def _plain_product(s):
    group = s['case']['group']
    w = s['w'].float() * s['scales'].float().repeat_interleave(group, 1)[:, :s['case']['k']]
    return torch.matmul(s['x'].float(), w.t()).to(s['x'].dtype)


def run(state):
    return globals()[('_own_' if own else '_plain_') + state['case']['op']](state)


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = {'case': case}
        globals()['_prepare_' + case['op']](case, seed, torch.Generator(device='cuda').manual_seed(seed), s)
        return globals()['_exact_' + case['op']](s)


def _exact_plan(s):
    """Request by request, as one would on paper."""
    c = s['case']
    page, cap = c['page'], s['tokens']
    lens, new, ring, table = (s[k].cpu().tolist() for k in ('lens', 'new', 'ring', 'table'))
    head, count = s['ring_state'].cpu().tolist()
    blocks, cu, slots, places = len(ring), [0], [], []
    begin, tail = head, head + count
    for i, n in enumerate(new):
        have = -(-lens[i] // page)
        if n < 0:
            for j in range(have):
                ring[tail % blocks] = table[i][j]
                tail += 1
            lens[i], n = 0, 0
        else:
            for j in range(have, -(-(lens[i] + n) // page)):
                table[i][j] = ring[head % blocks]
                head += 1
            for t in range(lens[i], lens[i] + n):
                slots.append(table[i][t // page] * page + t % page)
                places.append(t)
            lens[i] += n
        cu.append(cu[-1] + n)
    blank = [-1] * (cap - len(slots))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return {'lens': i32(lens), 'cu': i32(cu), 'slots': i32(slots + blank), 'places': i32(places + blank), 'ring_state': i32([head % blocks, tail - head]),
            'status': i32([0]), 'table': i32(table), 'ring': i32(ring)}


def _exact_append(s):
    c = s['case']
    h, kv, d, page, rot = c['heads'], c['kv_heads'], c['dim'], c['page'], c['rot']
    top = LARGEST[c['cache']]

    def turned(x):
        x = x.double()
        if rot:
            z = torch.view_as_complex(s['rope'][s['places'].long()].double())[:, None]
            z = z * torch.complex(x[..., :rot // 2], x[..., rot // 2:rot])
            x = torch.cat([z.real, z.imag, x[..., rot:]], -1)
        return x

    stored = (lambda x: torch.round(x)) if c['cache'] == 'int8' else (lambda x: x.to(torch.float8_e4m3fn).double())
    pool, scales, slots = s['pool'].double(), s['scales'].double(), s['slots'].cpu().numpy()
    new = [turned(s['k']), s['v'].double()]
    begin = 0
    while begin < len(slots):  # the tokens that go to one page, in order
        block, off = divmod(int(slots[begin]), page)
        end = begin + 1
        while end < len(slots) and int(slots[end]) // page == block:
            end += 1
        n = end - begin
        for which in (0, 1):
            x = new[which][begin:end].transpose(0, 1)  # [kv, n, d]
            was = pool[block, which].view((kv, page, d) if which == 0 else (kv, d, page))
            at = was if which == 0 else was.transpose(1, 2)
            least = x.abs().amax((1, 2)).clamp_min(FLOOR) / top
            if off:
                scale = torch.maximum(scales[block, which], least)
                at[:, :off] = stored(at[:, :off] * (scales[block, which] / scale)[:, None, None])
            else:
                scale = least
            at[:, off:off + n] = stored(x / scale[:, None, None])
            scales[block, which] = scale
        begin = end
    return [pool * scales[..., None], scales] + ([turned(s['q'])] if rot else [])


def _exact_attention(s):
    c = s['case']
    kv, d, page, group = c['kv_heads'], c['dim'], c['page'], c['heads'] // c['kv_heads']
    out, row = torch.empty((s['q'].shape[0], c['heads'], d), dtype=torch.float64, device='cuda'), 0
    for i, (past, new) in enumerate(zip(s['past'], s['new'])):
        n = past + new
        ids = s['table'][i, :_pages(n, page)].long()
        first = max(0, past + 1 - c['window']) if c['window'] else 0
        place = torch.arange(past, n, device='cuda').view(-1, 1, 1)
        at = torch.arange(first, n, device='cuda').view(1, 1, -1)
        hidden = at > place
        if c['window']:
            hidden = hidden | (place - at >= c['window'])
        for j in range(kv):
            k = (s['pool'][ids, 0, j].double() * s['scales'][ids, 0, j].double()[:, None]).view(-1, d)[first:n]
            v = (s['pool'][ids, 1, j].double() * s['scales'][ids, 1, j].double()[:, None]).view(-1, d, page).permute(0, 2, 1).reshape(-1, d)[first:n]
            q = s['q'][row:row + new, j * group:(j + 1) * group].double()
            z = (q.reshape(-1, d) @ k.t().contiguous()).view(new, group, -1) * d**-0.5
            z = z.masked_fill(hidden, -math.inf)
            z = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            out[row:row + new, j * group:(j + 1) * group] = (z.view(new * group, -1) @ v).view(new, group, d)
        row += new
    return out


def _exact_product(s):
    c = s['case']
    total = torch.zeros((c['rows'], c['n']), dtype=torch.float64, device='cuda')
    for j in range(s['scales'].shape[1]):
        a, b = j * c['group'], min(c['k'], (j + 1) * c['group'])
        total += (s['x'][:, a:b].double() @ s['w'][:, a:b].double().t().contiguous()) * s['scales'][:, j].double()
    return total
