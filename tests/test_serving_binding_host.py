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
