"""The attention's workspace holds whatever its last user left there: results are the same bits whatever that is, nothing is written around it."""
import numpy as np
import pytest
import torch

from tensorrt_llm.runtime import paged_kv8 as P
from test_gpu_serving_ops import check_attention

pytestmark = pytest.mark.gpu


class Filled:
    """Stands in for PagedKV8Cache._attend: a workspace of exactly the stated bytes, full of `value`, between two guards."""

    def __init__(self, value):
        self.value, self.used = value, 0

    def __call__(self, cache, p, stream):
        lib = P._lib()
        self.used = lib.tllm_paged_attention_workspace(p)
        assert self.used > 0 and self.used % 4 == 0
        room = torch.full((64 + self.used // 4 + 64, ), self.value, device='cuda')
        rc = lib.tllm_paged_attention(p, room[64:].data_ptr(), stream)
        same = room.view(torch.int32)
        assert (same[:64] == same[0]).all() and (same[-64:] == same[0]).all()
        return rc


# Tokens beside prompts, whose keys are split into a different number of parts each: more parts of the token's (by max_kv 19) than of the prompt's,
# as many, fewer; prompts of which one is no longer than a tile of rows of one head
@pytest.mark.parametrize('kind,dtype,size', [('int8', 'fp16', 128), ('fp8', 'bf16', 64), ('int8', 'bf16', 256)])
@pytest.mark.parametrize('kv,group,spans,max_kv', [(8, 4, [(900, 1), (700, 40)], 20000), (8, 4, [(300, 2), (0, 0), (700, 33)], 20000), (2, 1, [(2100, 1), (2500, 70), (40, 1)], 5000),
                                                   (2, 1, [(1200, 17), (1500, 20)], 40000), (1, 3, [(1700, 1), (3000, 1)], 9000)])
def test_attention_whatever_the_workspace_held(kv, group, spans, max_kv, kind, dtype, size, monkeypatch):
    got = []
    for value in (0.0, float('nan'), 1e30):
        fill = Filled(value)
        monkeypatch.setattr(P.PagedKV8Cache, '_attend', lambda cache, p, stream: fill(cache, p, stream))
        got.append(check_attention(np.random.default_rng(size + kv), kind, dtype, 64, size, kv, group, spans, max_kv=max_kv, spare_rows=1))
        assert fill.used
    assert all(np.array_equal(got[0], g) for g in got[1:])
