"""What the bindings of the serving operators do around the library's calls, without a GPU: a stand-in takes the library's place."""
import types
import weakref

import pytest
import torch

from tensorrt_llm.runtime import paged_kv8 as P


def test_the_workspace_lives_until_the_call_has_returned(monkeypatch):
    """A tensor that is dropped before the call goes back to torch's cache, from which another thread may take it between the call's launches."""
    made, seen, empty = [], [], torch.empty

    def watched(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append(weakref.ref(t))
        return t

    def attend(p, workspace, stream):
        held = made[-1]()
        seen.append(held is not None and held.data_ptr() == workspace)
        return 0

    monkeypatch.setattr(P, '_lib_', types.SimpleNamespace(tllm_paged_attention_workspace=lambda p: 4096, tllm_paged_attention=attend))
    monkeypatch.setattr(torch, 'empty', watched)
    cache = types.SimpleNamespace(pool=torch.zeros(1))
    assert P.PagedKV8Cache._attend(cache, b'', 0) == 0
    assert len(made) == 1 and seen == [True]
    assert made[0]() is None  # and no longer


def test_numbers_that_the_structures_do_not_hold_are_refused():
    """As every other wrong argument: a ValueError, and nothing is called."""
    cache = P.PagedKV8Cache.__new__(P.PagedKV8Cache)
    for name, v in dict(_index=-1, head_size=64, kv_heads=1, page_size=16, blocks=2, _type=2, _at=(64, 64), _attend=lambda p, stream: pytest.fail('called')).items():
        object.__setattr__(cache, name, v)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)
    q = torch.zeros((1, 1, 64), dtype=torch.float16)
    args = q, ints(0, 1).view(1, 2), ints(0, 1), ints(3)
    for bad in (dict(max_new=1 << 31), dict(max_new=1.5), dict(max_new=1, max_kv=1 << 40), dict(max_new=1, window=-(1 << 35)), dict(max_new=1, scale='1'), dict(max_new=None)):
        with pytest.raises(ValueError, match='argument'):
            cache.attention(*args, **bad)
