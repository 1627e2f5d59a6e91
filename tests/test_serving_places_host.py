"""Results of the serving operators that lie on other tensors are refused on the host, tensors beside or between each other are not: strided rows of one buffer are ordinary."""
import ctypes

import pytest
import torch

from tensorrt_llm.plugin import capi
from tensorrt_llm.runtime import paged_kv8 as P
from test_serving_api_host import AT, plan_params

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
