"""What the serving operators take at the ends of their ranges, asked of the library without a GPU."""
import ctypes

import pytest

from tensorrt_llm.plugin import capi
from tensorrt_llm.runtime import paged_kv8 as P
from test_serving_api_host import AT, attention_params


@pytest.mark.parametrize('n_seqs,n_rows,q_heads,kv_heads,size,max_new,fits', [
    (4096, 4095 + 8192, 64, 8, 128, 8192, True),     # tokens beside one long prompt
    (4096, 4095 + 16384, 32, 8, 128, 16384, True),
    (1, 1 << 19, 32, 32, 128, 1 << 19, True),        # one prompt of all rows
    (4096, 1 << 19, 64, 64, 64, 128, True),
    (4096, 4095 + 8192, 64, 8, 256, 8192, True),
    (4096, 4096, 64, 64, 128, 1 << 19, True),        # max_new beyond the rows that there are
    (4096, 1 << 19, 128, 8, 128, 1 << 19, False),
    (4096, 4095 + 8200, 64, 16, 256, 8200, False),
])
def test_attention_takes_every_batch_that_a_launch_holds(n_seqs, n_rows, q_heads, kv_heads, size, max_new, fits):
    p = attention_params()
    for name, v in dict(n_seqs=n_seqs, n_rows=n_rows, q_heads=q_heads, kv_heads=kv_heads, head_size=size, max_new=max_new, max_kv=100, q_row=q_heads * size, q_head=size, out_row=q_heads * size, out_head=size).items():
        setattr(p, name, v)
    got = P._lib().tllm_paged_attention_workspace(ctypes.addressof(p))
    assert (got >= 0) == fits, capi.last_error()
    if not fits:
        assert 'one launch' in capi.last_error()
