"""include/tllm_serving_api.h without a GPU: the entry points are exported, and refuse on the host, with a reason, what their kernels do not take; the
weights' packing is the documented layout; the oracle's own pieces agree with each other."""
import copy
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from oracle import serving_oracle as O
from tensorrt_llm.plugin import capi
from tensorrt_llm.quantization import group as G
from tensorrt_llm.runtime import paged_kv8 as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 1 << 20  # an address that nothing reads: every call here is refused first


def test_every_declared_entry_is_exported():
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'tllm_serving_api.h')).read(), flags=re.S)
    names = set(re.findall(r'\b(tllm_(?:paged|group)_\w+)\s*\(', text))
    assert names == {'tllm_paged_plan', 'tllm_paged_append', 'tllm_paged_attention_workspace', 'tllm_paged_attention', 'tllm_group_matmul'}
    lib = capi.load_library()
    assert all(hasattr(lib, n) for n in names)


i32, i64, ptr, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class PlanParams(ctypes.Structure):
    _fields_ = [(n, i32) for n in 'n_seqs n_rows page_size num_blocks max_blocks'.split()] + [('table_stride', i64)] + [
        (n, ptr) for n in 'lens new_lens ring ring_state block_table cu_tokens slot_map positions lens_out ring_state_out status'.split()]


class AppendParams(ctypes.Structure):
    _fields_ = [(n, i32) for n in 'n_rows kv_heads q_heads head_size page_size num_blocks dtype cache_type rot_dim rope_pairs rope_len'.split()] + [
        (n, ptr) for n in 'k v q q_out'.split()] + [(n, i64) for n in 'k_row k_head v_row v_head q_row q_head q_out_row q_out_head'.split()] + [
            (n, ptr) for n in 'slot_map positions rope pool scales'.split()]


class AttentionParams(ctypes.Structure):
    _fields_ = [(n, i32) for n in 'n_seqs n_rows q_heads kv_heads head_size page_size num_blocks max_blocks dtype cache_type max_new max_kv window'.split()] + [
        ('scale', f32)] + [(n, i64) for n in 'table_stride q_row q_head out_row out_head'.split()] + [
            (n, ptr) for n in 'q pool scales block_table cu_tokens kv_lens out'.split()]


class MatmulParams(ctypes.Structure):
    _fields_ = [(n, i32) for n in 'rows n k group dtype'.split()] + [('ldx', i64), ('ldy', i64)] + [(n, ptr) for n in 'x packed scales y'.split()]


def test_the_binding_lays_out_what_the_header_declares():
    """Field by field in the header's order, and as large as C has them."""
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'tllm_serving_api.h')).read(), flags=re.S)
    for mine, packed, name in ((PlanParams, P._PLAN, 'paged_plan'), (AppendParams, P._APPEND, 'paged_append'), (AttentionParams, P._ATTENTION, 'paged_attention'),
                               (MatmulParams, G._PARAMS, 'group_matmul')):
        body = re.search(r'typedef struct\s*\{([^}]*)\}\s*tllm_%s_params_t;' % name, text).group(1)
        fields = []
        for kind, star, names in re.findall(r'(?:const\s+)?(void|int32_t|int64_t|float)\s*(\*?)\s*([\w,\s]+);', body):
            fields += [(n.strip(), ptr if star else {'int32_t': i32, 'int64_t': i64, 'float': f32}[kind]) for n in names.split(',')]
        assert fields == mine._fields_ and packed.size == ctypes.sizeof(mine)
        codes = ''.join(int(n or 1) * c for n, c in re.findall(r'(\d*)([a-zA-Z])', packed.format))
        assert codes == ''.join({i32: 'i', i64: 'q', f32: 'f', ptr: 'P'}[t] for _, t in fields)


def refused(call, params, word, **bad):
    p = type(params)()
    ctypes.memmove(ctypes.addressof(p), ctypes.addressof(params), ctypes.sizeof(p))
    for k, v in bad.items():
        setattr(p, k, v)
    assert call(p) != 0 and word in capi.last_error(), (bad, capi.last_error())


def plan_params():
    p = PlanParams(4, 8, 16, 100, 5, 5)
    for n, _ in p._fields_[6:]:
        setattr(p, n, AT)
    return p


def test_plan_refuses():
    lib = P._lib()
    call = lambda p: lib.tllm_paged_plan(ctypes.addressof(p), None)
    assert lib.tllm_paged_plan(None, None) != 0
    p = plan_params()
    for word, bad in (('n_seqs', dict(n_seqs=0)), ('n_seqs', dict(n_seqs=4097)), ('n_rows', dict(n_rows=-1)), ('n_rows', dict(n_rows=(1 << 19) + 1)), ('page_size', dict(page_size=0)),
                      ('page_size', dict(page_size=256)), ('page_size', dict(page_size=17)), ('num_blocks', dict(num_blocks=0)), ('num_blocks', dict(num_blocks=1 << 27)),
                      ('max_blocks', dict(max_blocks=0)), ('table_stride', dict(table_stride=4)), ('null', dict(lens=None)), ('null', dict(ring=None)), ('null', dict(slot_map=None)),
                      ('null', dict(status=None)), ('aligned', dict(positions=AT + 2)), ('aligned', dict(lens_out=AT + 1))):
        refused(call, p, word, **bad)


def test_plan_refuses_results_on_other_tensors():
    lib = P._lib()
    call = lambda p: lib.tllm_paged_plan(ctypes.addressof(p), None)
    p = plan_params()
    for i, (n, _) in enumerate(p._fields_[6:]):
        setattr(p, n, AT * (i + 1))
    for bad in (dict(lens_out=p.new_lens), dict(lens_out=p.lens + 4), dict(ring_state_out=p.ring_state + 4), dict(cu_tokens=p.lens), dict(slot_map=p.positions), dict(status=p.cu_tokens + 16),
                dict(positions=p.ring + 396), dict(lens_out=p.ring_state), dict(ring_state_out=p.lens)):
        refused(call, p, 'lies where', **bad)


def append_params():
    p = AppendParams(8, 2, 4, 64, 16, 100, capi.HALF, capi.INT8, 64, 0, 50)
    for n, t in p._fields_:
        if t is ctypes.c_void_p:
            setattr(p, n, AT)
        elif t is ctypes.c_int64:
            setattr(p, n, 64)
    return p


def test_append_refuses():
    lib = P._lib()
    call = lambda p: lib.tllm_paged_append(ctypes.addressof(p), None)
    assert lib.tllm_paged_append(None, None) != 0
    p = append_params()
    for word, bad in (('n_rows', dict(n_rows=-1)), ('dtype', dict(dtype=capi.FLOAT)), ('cache_type', dict(cache_type=capi.HALF)), ('head_size', dict(head_size=96)),
                      ('head_size', dict(head_size=32)), ('page_size', dict(page_size=8)), ('num_blocks', dict(num_blocks=0)), ('num_blocks', dict(num_blocks=1 << 28)),
                      ('kv_heads', dict(kv_heads=0)), ('pool', dict(pool=None)), ('pool', dict(pool=AT + 8)), ('scales', dict(scales=AT + 2)), ('q_heads', dict(q_heads=-1)),
                      ('rot_dim', dict(rot_dim=80)), ('rot_dim', dict(rot_dim=8)), ('rot_dim', dict(rot_dim=-16)), ('rope_pairs', dict(rope_pairs=2)), ('rope', dict(rope=None)),
                      ('rope', dict(rope_len=0)), ('rotated', dict(rot_dim=0)), ('slot map', dict(slot_map=None)), ('positions', dict(positions=None)), ('k has', dict(k=AT + 2)),
                      ('null v', dict(v=None)), ('v has', dict(v_row=65)), ('k has', dict(k_head=4)), ('q has', dict(q=AT + 8)), ('null q_out', dict(q_out=None))):
        refused(call, p, word, **bad)


def attention_params():
    p = AttentionParams(3, 8, 4, 2, 64, 16, 100, 7, capi.HALF, capi.INT8, 4, 100, 0, 0.125, 7)
    for n, t in p._fields_[15:]:
        setattr(p, n, AT if t is ctypes.c_void_p else 64)
    return p


def test_attention_refuses():
    lib = P._lib()
    call = lambda p: lib.tllm_paged_attention(ctypes.addressof(p), AT, None)
    assert lib.tllm_paged_attention(None, None, None) != 0
    p = attention_params()
    for word, bad in (('n_seqs', dict(n_seqs=0)), ('n_rows', dict(n_rows=-2)), ('q_heads', dict(q_heads=3)), ('q_heads', dict(q_heads=0)), ('kv_heads', dict(kv_heads=0)),
                      ('head_size', dict(head_size=80)), ('page_size', dict(page_size=4)), ('max_blocks', dict(max_blocks=0)), ('table_stride', dict(table_stride=6)),
                      ('dtype', dict(dtype=capi.INT8)), ('cache_type', dict(cache_type=capi.UINT8)), ('max_new', dict(max_new=0)), ('max_kv', dict(max_kv=-1)), ('window', dict(window=-1)),
                      ('scale', dict(scale=float('nan'))), ('scale', dict(scale=float('inf'))), ('null', dict(block_table=None)), ('null', dict(cu_tokens=None)), ('aligned', dict(kv_lens=AT + 1)),
                      ('q has', dict(q=AT + 2)), ('q has', dict(q_row=63)), ('out has', dict(out_head=9)), ('null out', dict(out=None)),
                      ('one launch', dict(n_seqs=4096, max_new=1 << 19, n_rows=1 << 19))):
        refused(call, p, word, **bad)
    assert lib.tllm_paged_attention_workspace(None) == -1
    p.max_new = 0
    assert lib.tllm_paged_attention_workspace(ctypes.addressof(p)) == -1


def test_matmul_refuses():
    call = lambda p: G._entry()(ctypes.addressof(p), None)
    assert G._entry()(None, None) != 0
    p = MatmulParams(2, 10, 64, 32, capi.HALF, 64, 10, AT, AT, AT, AT)
    for word, bad in (('dtype', dict(dtype=capi.FLOAT)), ('group', dict(group=16)), ('rows', dict(rows=-1)), ('k 48', dict(k=48)), ('k 0', dict(k=0)), ('n 0', dict(n=0)),
                      ('weights', dict(packed=None)), ('weights', dict(packed=AT + 8)), ('scales', dict(scales=AT + 2)), ('x has', dict(x=AT + 2)), ('x has', dict(ldx=63)), ('x has', dict(ldx=32)),
                      ('y is', dict(y=None)), ('y is', dict(ldy=9)), ('y lies', dict())):
        refused(call, p, word, **bad)


@pytest.mark.parametrize('n,k,group', [(1, 32, 32), (21, 160, 64), (33, 288, 128)])
def test_packing_is_the_documented_layout(n, k, group):
    g = torch.Generator().manual_seed(n)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    s = torch.rand((n, -(-k // group)), generator=g).half()
    packed, scales = (t.numpy() for t in G.pack(q, s, group))
    assert packed.shape == (-(-n // 16), -(-k // 128), 64, 16) and scales.shape == (-(-k // group), -(-n // 16) * 16)
    order = [0, 2, 4, 6, 1, 3, 5, 7]
    words = packed.view('<u4')
    for row in range(packed.shape[0] * 16):
        for col in range(packed.shape[1] * 128):
            j, e8 = divmod(col % 128, 32)
            nibble = words[row // 16, col // 128, 16 * (e8 // 8) + row % 16, j] >> (4 * order.index(e8 % 8)) & 15
            assert nibble == (int(q[row, col]) + 8 if row < n and col < k else 8)
    assert np.array_equal(scales[:, :n], s.t().numpy()) and not scales[:, n:].any()


def test_packing_refuses():
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2).half()
    for bad in ((q, s, 16), (q[:, :48].contiguous(), s, 32), (q.int(), s, 32), (q, s.float(), 32), (q, s[:, :1], 32), (q + 8, s, 32), (q - 9, s, 32)):
        with pytest.raises(ValueError):
            G.pack(*bad)
    with pytest.raises(ValueError):
        G.GroupQuantMatmul(q, s, 32)  # not on a GPU


def test_quantize():
    w = torch.linspace(-3, 3, 5 * 96).view(5, 96)
    w[1] = 0
    q, s = G.quantize(torch.nn.Parameter(w), 64)
    assert q.shape == (5, 96) and s.shape == (5, 2) and not s.requires_grad and int(q.min()) >= -8 and int(q.max()) <= 7 and (s[1] == 1).all() and (q[1] == 0).all()
    # half a step, and what the scale's rounding (2^-11) moves 7 steps by
    assert ((q.float() * s.float().repeat_interleave(64, 1)[:, :96] - w).abs() <= (0.5 + 7 * 2.0**-11) * s.float().repeat_interleave(64, 1)[:, :96]).all()
    for bad in (float('inf'), float('nan'), 1e6):
        x = w.clone()
        x[2, 70] = bad
        with pytest.raises(ValueError, match='finite'):
            G.quantize(x, 64)


def test_public_names():
    import tensorrt_llm.quantization as Q
    import tensorrt_llm.runtime as R
    assert Q.GroupQuantMatmul is G.GroupQuantMatmul and R.PagedKV8Cache is P.PagedKV8Cache and R.plan_step is P.plan_step and R.StepPlan is P.StepPlan
    assert R.DeviceBlockPool is P.DeviceBlockPool and R.rope_table is P.rope_table
    for module in (Q, R):
        with pytest.raises(AttributeError):
            module.no_such_name


def test_caches_and_pools_refuse():
    pool, scales = torch.zeros((3, 2, 2, 16 * 64), dtype=torch.int8), torch.zeros((3, 2, 2))
    for bad in ((pool, scales, 16, 64), (pool, scales, 16, 128), (pool, scales, 24, 64), (pool.float(), scales, 16, 64), (pool, scales[:2], 16, 64), (pool[..., ::2], scales, 16, 64)):
        with pytest.raises(ValueError):
            P.PagedKV8Cache(*bad)
    for bad in ((0, 16, 1, 1), (4, 20, 1, 1), (4, 16, 0, 1), (4, 16, 1, 0), (1 << 28, 16, 1, 1)):
        with pytest.raises(ValueError):
            P.DeviceBlockPool(*bad, device='cpu')
    b = P.DeviceBlockPool(4, 16, 2, 3, device='cpu')
    with pytest.raises(ValueError, match='GPU'):
        b.plan(torch.tensor([1, 1], dtype=torch.int32), 2)
    for other in (dict(), dict(lens=b.lens), dict(ring_state=b.ring_state)):  # it would leave the pool's own state behind
        with pytest.raises(ValueError, match='over this pool'):
            b.plan(torch.tensor([1, 1], dtype=torch.int32), 2, P.StepPlan(2, 2, 'cpu', **other))
    with pytest.raises(TypeError, match='copied'):
        copy.copy(P.StepPlan(2, 2, 'cpu'))


def test_the_oracle_keeps_what_it_is_given():
    """Its cache gives back what was appended within its steps, whether at once or token by token, and its plans lose no block."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 2, 64)).astype(np.float32)
    slots = np.arange(5, 45)
    for kind, most in (('int8', lambda v, s: 0.5001 * s), ('fp8', lambda v, s: 2.0**-4 * np.abs(v) * 1.0001 + 2.0**-10 * s)):
        pool, scales = np.zeros((3, 2, 2, 16 * 64), np.float32), np.ones((3, 2, 2), np.float32) * 1e-3
        O.append(pool, scales, x, x, slots, 16, kind, 65504)
        keys = pool[:, 0].reshape(3, 2, 16, 64).transpose(0, 2, 1, 3).reshape(48, 2, 64)[5:45]
        vals = pool[:, 1].reshape(3, 2, 64, 16).transpose(0, 3, 1, 2).reshape(48, 2, 64)[5:45]
        s = scales[slots // 16].transpose(0, 2, 1)[..., None, :]  # [rows, heads, 1, 2]
        assert (np.abs(keys * s[..., 0] - x) <= most(x, s[..., 0])).all() and (np.abs(vals * s[..., 1] - x) <= most(x, s[..., 1])).all()
    p = O.plan([16, 3, 40], [1, -1, 9], np.array([9, 8, 7, 0, 0, 0, 0, 0, 0, 0]), [0, 3], np.array([[1, 0, 0, 0], [2, 0, 0, 0], [3, 4, 5, 0]]), 16, 12)
    assert p['status'] == 0 and p['table'].tolist() == [[1, 9, 0, 0], [2, 0, 0, 0], [3, 4, 5, 8]] and p['state'] == [2, 2] and p['ring'][2:4].tolist() == [7, 2]
    assert p['lens'] == [17, 0, 49] and p['cu'] == [0, 1, 1, 10] and p['slots'][:4] == [144, 5 * 16 + 8, 5 * 16 + 9, 5 * 16 + 10] and p['slots'][9] == 128
