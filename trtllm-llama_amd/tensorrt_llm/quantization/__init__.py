from .mode import QuantMode

__all__ = ['QuantMode', 'GroupQuantMatmul']


def __getattr__(name):
    if name == 'GroupQuantMatmul':  # it brings torch in, which the mode does without
        from .group import GroupQuantMatmul
        return GroupQuantMatmul
    raise AttributeError(f'module {__name__!r} has no attribute {name!r}')
