"""Results of the serving operators that lie on other tensors are refused on the host, tensors beside or between each other are not: strided rows of one buffer are ordinary."""
import ctypes

import pytest
import torch

from tensorrt_llm.plugin import capi
from tensorrt_llm.quantization import group as G
from tensorrt_llm.runtime import paged_kv8 as P
from test_serving_api_host import AT, AppendParams, MatmulParams, attention_params, plan_params

# a call that passes the checks ends at the launch, which there has to be no device for: its addresses are made up
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason='the addresses are no memory')


def plan_places():
    """Every tensor in a mebibyte of its own."""
    p = plan_params()
    for i, (n, _) in enumerate(p._fields_[6:]):
        setattr(p, n, AT * (i + 1))
    return p


def refused(call, p, word, **bad):
    q = type(p).from_buffer_copy(p)
    for k, v in bad.items():
        setattr(q, k, v)
    rc = call(q)
    return rc != 0 and word in capi.last_error()


@pytest.mark.parametrize('bad', [dict(block_table='lens'), dict(block_table='new_lens'), dict(block_table='ring'), dict(block_table='slot_map', max_blocks=5), dict(block_table='lens_out'),
                                 dict(ring='lens'), dict(ring='new_lens'), dict(ring='ring_state'), dict(ring='status'), dict(block_table='cu_tokens', table_stride=1 << 16),
                                 dict(block_table=-4, table_stride=100)], ids=str)
def test_plan_refuses_tables_and_rings_on_other_tensors(bad):
    p = plan_places()
    bad = {k: getattr(p, v) if isinstance(v, str) else v for k, v in bad.items()}
    if bad.get('block_table') == -4:  # the second of the table's rows begins behind the lengths' first 12 bytes
        bad['block_table'] = p.lens + 12 - 400
    assert refused(lambda q: P._lib().tllm_paged_plan(ctypes.addressof(q), None), p, 'lies where', **bad)


# whether a vector meets strided rows, against sets of places
@pytest.mark.parametrize('stride', [5, 6, 9, 16, 31])
def test_plan_finds_every_place_in_a_table(stride):
    p = plan_places()
    p.table_stride, base = stride, p.block_table
    table = {base + 4 * (r * stride + c) for r in range(p.n_seqs) for c in range(p.max_blocks)}
    for word in range(-8, p.n_seqs * stride + 8):
        lens = {base + 4 * (word + i) for i in range(p.n_seqs)}
        assert refused(lambda q: P._lib().tllm_paged_plan(ctypes.addressof(q), None), p, 'lies where', new_lens=base + 4 * word) == bool(lens & table), word


def matmul(**with_):
    p = MatmulParams(8, 24, 64, 32, capi.HALF, 64, 24, AT, 4 * AT, 5 * AT, 2 * AT)
    for k, v in with_.items():
        setattr(p, k, v)
    return G._entry()(ctypes.addressof(p), None) != 0 and 'y lies' in capi.last_error()


def test_products_refuse_results_on_their_operands():
    assert not matmul()
    assert matmul(y=AT) and matmul(y=AT + 2 * 64 * 8 - 2) and not matmul(y=AT + 2 * 64 * 8) and matmul(y=AT - 2 * 24 * 8 + 2) and not matmul(y=AT - 2 * 24 * 8)
    assert matmul(y=4 * AT + 2) and matmul(y=5 * AT + 2 * 32 * 2 - 2) and not matmul(y=5 * AT + 2 * 32 * 2)  # 2 tiles of 16 outputs, one k-tile; 2 groups of 32 scales
    # rows of one buffer: y behind x, y before x, y across x
    for ld in (88, 96, 200):
        assert not matmul(ldx=ld, ldy=ld, y=AT + 128) and not matmul(ldx=ld, ldy=ld, y=AT - 48)
        assert matmul(ldx=ld, ldy=ld, y=AT + 126) and matmul(ldx=ld, ldy=ld, y=AT - 46)
        assert matmul(ldx=ld, ldy=ld, y=AT + 128 + 14 * ld) is False and matmul(ldx=ld, ldy=ld, y=AT + 126 + 14 * ld)  # seven rows on
    assert matmul(rows=1, y=AT + 126) and not matmul(rows=1, y=AT + 128)


def test_products_of_rows_of_any_two_strides_against_sets_of_places():
    for ldx, ldy, rows in ((64, 24, 5), (72, 40, 6), (128, 136, 4), (200, 24, 3)):
        x = {2 * (r * ldx + c) for r in range(rows) for c in range(64)}
        for first in range(-2 * rows * ldy - 64, 2 * rows * ldx + 64, 10):
            y = {first + 2 * (r * ldy + c) for r in range(rows) for c in range(24)}
            assert matmul(rows=rows, ldx=ldx, ldy=ldy, y=AT + first) == bool(x & y), (ldx, ldy, first)


def append(**with_):
    """Rows of 4 heads of queries, 2 of keys and 2 of values, packed; q_out far from them."""
    p = AppendParams(8, 2, 4, 64, 16, 100, capi.HALF, capi.INT8, 64, 0, 50)
    at = dict(q=AT, k=AT + 512, v=AT + 768, q_out=2 * AT, slot_map=3 * AT, positions=4 * AT, rope=5 * AT, pool=6 * AT, scales=9 * AT, q_out_row=256)
    for n in ('k', 'v', 'q', 'q_out'):
        at.setdefault(n + '_row', 512)
        at[n + '_head'] = 64
    for n, v in {**at, **with_}.items():
        setattr(p, n, v)
    rc = P._lib().tllm_paged_append(ctypes.addressof(p), None)
    assert rc != 0 or p.n_rows == 0
    return 'q_out lie' in capi.last_error()


def test_append_refuses_queries_on_other_rows():
    assert not append() and not append(q_out=AT, q_out_row=512)
    assert append(q_out=AT) and append(q_out=AT + 16, q_out_row=512) and append(q_out=AT + 512, q_out_row=512) and append(q_out=AT + 768, q_out_row=512)
    assert append(q_out=AT + 1024, q_out_row=1024) and not append(q_out=AT + 1024, q_out_row=1024, q_row=1024, k_row=1024, v_row=1024)  # every second row of a buffer
    assert append(q_out_row=64) and append(q_out_row=0) and append(q_out_head=0) and append(q_out_head=32) and not append(q_out_row=64, q_out_head=512)
    assert append(q_out_row=-128) and not append(q_out=2 * AT + 1 * AT // 2, q_out_row=-256)


def attention(**with_):
    p = attention_params()
    at = dict(q=AT, q_row=256, q_head=64, out=2 * AT, out_row=256, out_head=64, block_table=3 * AT, cu_tokens=4 * AT, kv_lens=5 * AT, pool=6 * AT, scales=9 * AT)
    for n, v in {**at, **with_}.items():
        setattr(p, n, v)
    return P._lib().tllm_paged_attention_workspace(ctypes.addressof(p)) == -1 and ('out lie' in capi.last_error())


def test_attention_refuses_results_on_queries():
    assert not attention() and not attention(out=AT)
    assert attention(out=AT + 16) and attention(out=AT, out_row=512) and attention(out=AT + 2 * 256 * 8 - 16) and not attention(out=AT + 2 * 256 * 8)
    assert attention(out_row=64) and attention(out_head=8) and attention(out_row=248)
    assert not attention(n_rows=1, max_new=1, out=AT, out_row=0) and attention(n_rows=1, max_new=1, out=AT + 256)


def test_attention_finds_rows_and_heads_of_any_strides_against_sets_of_places():
    """Places in units of 16 bytes, which all addresses and strides are multiples of."""
    def places(at, row, head):
        return {at + r * row + h * head + e for r in range(3) for h in range(2) for e in range(8)}

    shapes = [(16, 8), (40, 16), (48, 24), (8, 24), (8, 32), (24, 8), (56, 8), (21, 40), (-16, 8), (40, -16)]
    for q_row, q_head in shapes:
        q = places(0, q_row, q_head)
        for row, head in shapes:
            for at in range(-130, 130):
                out = places(at, row, head)
                want = len(out) < 48 or bool(out & q) and not (at == 0 and (row, head) == (q_row, q_head))
                got = attention(n_rows=3, q_heads=2, kv_heads=1, q_row=q_row * 8, q_head=q_head * 8, out=AT + 16 * at, out_row=row * 8, out_head=head * 8)
                assert got == want, ((q_row, q_head), (row, head), at)
