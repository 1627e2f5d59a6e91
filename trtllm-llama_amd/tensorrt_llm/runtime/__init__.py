from .generation import GenerationSession, ModelConfig, RaggedGenerationSession, SamplingConfig
from .kv_cache_manager import GenerationSequence, KVCacheManager, StateSlotManager
from .scheduler import RaggedScheduler, Request
from .session import Session, TensorInfo

__all__ = ['ModelConfig', 'GenerationSession', 'RaggedGenerationSession', 'RaggedScheduler', 'Request', 'StateSlotManager', 'GenerationSequence', 'KVCacheManager', 'SamplingConfig', 'Session',
           'TensorInfo', 'DeviceBlockPool', 'PagedKV8Cache', 'StepPlan', 'plan_step', 'rope_table']


def __getattr__(name):
    if name in ('DeviceBlockPool', 'PagedKV8Cache', 'StepPlan', 'plan_step', 'rope_table'):  # they bring torch in, which the sessions do without
        from . import paged_kv8
        return getattr(paged_kv8, name)
    raise AttributeError(f'module {__name__!r} has no attribute {name!r}')
