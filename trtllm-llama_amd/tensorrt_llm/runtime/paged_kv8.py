"""Pages, an 8-bit cache and its attention for steps over packed batches (ctypes binding of include/tllm_serving_api.h).

Where KVCacheManager hands out block ids on the host, `DeviceBlockPool` keeps the free list, the tables and the lengths on the GPU: one
`plan` a step serves every layer, and nothing of it comes back to the host, so a step with it can be captured into a graph.  `PagedKV8Cache` is one
layer's cache: int8 or e4m3 elements (torch.int8, torch.float8_e4m3fn) under a scale for each page and head, filled by `append` and read by
`attention`.  Tensors are handed over as device pointers; calls run on torch's current stream of the tensors' device and check their
arguments (TypeError, ValueError; RuntimeError with the library's reason).  A failing call has launched nothing."""
import ctypes
import math
from typing import Optional

import torch

from ..plugin import capi

BF16 = 7
PAGE_SIZES, HEAD_SIZES = (16, 32, 64, 128), (64, 128, 256)
_ACT = {torch.float16: capi.HALF, torch.bfloat16: BF16}
_CACHE = {torch.int8: capi.INT8, torch.float8_e4m3fn: capi.FP8}

_i32, _i64, _ptr, _f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class _PlanParams(ctypes.Structure):
    _fields_ = [(n, _i32) for n in ('n_seqs', 'n_rows', 'page_size', 'num_blocks', 'max_blocks')] + [('table_stride', _i64)] + [
        (n, _ptr) for n in ('lens', 'new_lens', 'ring', 'ring_state', 'block_table', 'cu_tokens', 'slot_map', 'positions', 'lens_out',
                            'ring_state_out', 'status')]


class _AppendParams(ctypes.Structure):
    _fields_ = [(n, _i32) for n in ('n_rows', 'kv_heads', 'q_heads', 'head_size', 'page_size', 'num_blocks', 'dtype', 'cache_type', 'rot_dim',
                                    'rope_pairs', 'rope_len')] + [(n, _ptr) for n in ('k', 'v', 'q', 'q_out')] + [
                                        (n, _i64) for n in ('k_row', 'k_head', 'v_row', 'v_head', 'q_row', 'q_head', 'q_out_row', 'q_out_head')
                                    ] + [(n, _ptr) for n in ('slot_map', 'positions', 'rope', 'pool', 'scales')]


class _AttentionParams(ctypes.Structure):
    _fields_ = [(n, _i32) for n in ('n_seqs', 'n_rows', 'q_heads', 'kv_heads', 'head_size', 'page_size', 'num_blocks', 'max_blocks', 'dtype',
                                    'cache_type', 'max_new', 'max_kv', 'window')] + [('scale', _f32)] + [
                                        (n, _i64) for n in ('table_stride', 'q_row', 'q_head', 'out_row', 'out_head')
                                    ] + [(n, _ptr) for n in ('q', 'pool', 'scales', 'block_table', 'cu_tokens', 'kv_lens', 'out')]


_lib_ = None


def _lib():
    global _lib_
    if _lib_ is None:
        lib = capi.load_library()
        for name in ('tllm_paged_plan', 'tllm_paged_append'):
            f = getattr(lib, name)
            f.argtypes, f.restype = [_ptr, _ptr], _i32
        lib.tllm_paged_attention.argtypes, lib.tllm_paged_attention.restype = [_ptr, _ptr, _ptr], _i32
        lib.tllm_paged_attention_workspace.argtypes, lib.tllm_paged_attention_workspace.restype = [_ptr], _i64
        _lib_ = lib
    return _lib_


def _raise(name):
    raise RuntimeError(f'{name}: {capi.last_error()}')


class _on(object):
    """The device of `t` is the current one while a call is issued."""
    __slots__ = ('index', 'back')

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *a):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _ints(what, t, n, device):
    """`t` is a contiguous int32 tensor of n values (n None: any number) on `device`."""
    if t.dtype is not torch.int32 or t.dim() != 1 or (n is not None and t.numel() != n) or not t.is_contiguous() or t.device != device:
        raise ValueError(f'{what} has to be a contiguous int32 vector{"" if n is None else f" of {n} values"} on {device}: got '
                         f'{t.dtype} {tuple(t.shape)} on {t.device}')
    return t.data_ptr()


def _table(t, rows, device):
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] < rows or t.shape[1] < 1 or t.stride(1) != 1 or t.device != device:
        raise ValueError(f'block_table has to be int32 [{rows} or more, blocks] with contiguous rows on {device}: got {t.dtype} {tuple(t.shape)} on {t.device}')
    return t.data_ptr()


def _rows(what, t, rows, heads, size, dtype, device):
    """`t` is [rows, heads, size] of `dtype` with a contiguous last dimension; views into packed projections are fine."""
    if t.dtype is not dtype or t.dim() != 3 or t.shape[2] != size or t.shape[0] != rows or (heads is not None and t.shape[1] != heads) \
            or t.device != device or t.stride(2) != 1:
        raise ValueError(f'{what} has to be {dtype} [{rows}, {"heads" if heads is None else heads}, {size}] with a contiguous last dimension on {device}: '
                         f'got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}')
    return t.data_ptr()


def _strides(t, written=False):
    """Row and head strides; of a dimension of one they say nothing."""
    row, head = t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2], t.stride(1) if t.shape[1] > 1 else t.shape[2]
    if written and min(row, head) < t.shape[2]:
        raise ValueError(f'rows that are written overlap: strides {t.stride()}')
    return row, head


def _table_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class StepPlan(object):
    """What a step needs to know of its pages, in tensors that are written anew by every plan: cu_tokens [n_seqs + 1], slot_map and positions [n_rows]
    (-1 behind the last row), lens [n_seqs] and ring_state [2] behind the step, status [1] (0: fine; tllm_serving_api.h has the others)."""

    def __init__(self, n_seqs: int, n_rows: int, device, lens: Optional[torch.Tensor] = None, ring_state: Optional[torch.Tensor] = None):
        new = lambda n: torch.empty(n, dtype=torch.int32, device=device)
        self.cu_tokens, self.slot_map, self.positions, self.status = new(n_seqs + 1), new(n_rows), new(n_rows), new(1)
        self.lens = new(n_seqs) if lens is None else lens
        self.ring_state = new(2) if ring_state is None else ring_state


def plan_step(lens: torch.Tensor, new_lens: torch.Tensor, ring: torch.Tensor, ring_state: torch.Tensor, block_table: torch.Tensor, page_size: int,
              n_rows: int, out: Optional[StepPlan] = None) -> StepPlan:
    """Pages for the step's tokens (tllm_paged_plan): lens and new_lens int32 [n], a negative new length ends a request.  `block_table` and `ring`
    are updated; the lengths and the ring's state behind the step are out.lens and out.ring_state, which may be `lens` and `ring_state`."""
    device, n = lens.device, lens.numel()
    if out is None:
        out = StepPlan(n, n_rows, device)
    table = _table(block_table, n, device)
    p = _PlanParams(n, n_rows, page_size, ring.numel(), block_table.shape[1], _table_stride(block_table), _ints('lens', lens, None, device),
                    _ints('new_lens', new_lens, n, device), _ints('ring', ring, None, device), _ints('ring_state', ring_state, 2, device), table,
                    _ints('out.cu_tokens', out.cu_tokens, n + 1, device), _ints('out.slot_map', out.slot_map, n_rows, device),
                    _ints('out.positions', out.positions, n_rows, device), _ints('out.lens', out.lens, n, device),
                    _ints('out.ring_state', out.ring_state, 2, device), _ints('out.status', out.status, 1, device))
    if device.type != 'cuda':
        raise ValueError(f'the tensors have to be on a GPU: got {device}')
    with _on(lens) as stream:
        if _lib().tllm_paged_plan(ctypes.addressof(p), stream):
            _raise('plan_step')
    return out


class DeviceBlockPool(object):
    """`blocks` blocks of `page_size` tokens, shared by all layers, for at most `max_seqs` requests of at most `max_blocks` blocks: the free list, the
    requests' tables and lengths, all on the GPU.  A request is a row of the table; a row of length 0 is free for the next one."""

    def __init__(self, blocks: int, page_size: int, max_seqs: int, max_blocks: int, device='cuda'):
        if page_size not in PAGE_SIZES:
            raise ValueError(f'page_size is one of {PAGE_SIZES}: got {page_size}')
        if blocks < 1 or max_seqs < 1 or max_blocks < 1 or blocks * page_size >= 1 << 31:
            raise ValueError('blocks, max_seqs and max_blocks have to be positive, and blocks * page_size below 2^31')
        self.page_size, self.blocks, self.max_seqs, self.max_blocks = page_size, blocks, max_seqs, max_blocks
        self.ring = torch.arange(blocks, dtype=torch.int32, device=device)
        self.ring_state = torch.tensor([0, blocks], dtype=torch.int32, device=device)
        self.block_table = torch.zeros((max_seqs, max_blocks), dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)

    def plan(self, new_lens: torch.Tensor, n_rows: int, out: Optional[StepPlan] = None) -> StepPlan:
        """The next step: new_lens int32 [max_seqs] tokens that each request brings (0: none, negative: it ends and gives its blocks back), `n_rows`
        rows of the packed batch.  Lengths and free list are updated in place; out.lens is self.lens.  A step that does not fit changes
        nothing and says why in out.status; as it has no rows, what the step launches behind it touches nothing."""
        if out is None:
            out = StepPlan(self.max_seqs, n_rows, self.lens.device, lens=self.lens, ring_state=self.ring_state)
        return plan_step(self.lens, new_lens, self.ring, self.ring_state, self.block_table, self.page_size, n_rows, out)


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, factor: float = 1.0, device='cuda') -> torch.Tensor:
    """fp32 [positions, rot_dim / 2, 2]: cos and sin of position / factor * base^(-2 i / rot_dim), the angles formed in 64 bits."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / factor * base**(-2.0 * i / rot_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).to(device)


class PagedKV8Cache(object):
    """One layer's cache: `pool` int8 or float8_e4m3fn [blocks, 2, kv_heads, page_size * head_size] (keys of a page and head [page_size, head_size],
    values [head_size, page_size]) and `scales` fp32 [blocks, 2, kv_heads].  The tensors are the caller's; `PagedKV8Cache.empty` makes them."""

    def __init__(self, pool: torch.Tensor, scales: torch.Tensor, page_size: int, head_size: int):
        if page_size not in PAGE_SIZES or head_size not in HEAD_SIZES:
            raise ValueError(f'page_size is one of {PAGE_SIZES} and head_size one of {HEAD_SIZES}: got {page_size}, {head_size}')
        if pool.dtype not in _CACHE or pool.dim() != 4 or pool.shape[1] != 2 or pool.shape[3] != page_size * head_size or not pool.is_contiguous():
            raise ValueError(f'the pool has to be contiguous int8 or float8_e4m3fn [blocks, 2, kv_heads, {page_size * head_size}]: got {pool.dtype} {tuple(pool.shape)}')
        if scales.dtype is not torch.float32 or scales.shape != pool.shape[:3] or not scales.is_contiguous() or scales.device != pool.device:
            raise ValueError(f'the scales have to be contiguous float32 {tuple(pool.shape[:3])} on {pool.device}: got {scales.dtype} {tuple(scales.shape)} on {scales.device}')
        if pool.device.type != 'cuda':
            raise ValueError(f'the cache has to be on a GPU: got {pool.device}')
        self.pool, self.scales, self.page_size, self.head_size = pool, scales, page_size, head_size
        self.blocks, self.kv_heads, self._type = pool.shape[0], pool.shape[2], _CACHE[pool.dtype]

    @classmethod
    def empty(cls, blocks: int, page_size: int, kv_heads: int, head_size: int, dtype=torch.int8, device='cuda') -> 'PagedKV8Cache':
        return cls(torch.zeros((blocks, 2, kv_heads, page_size * head_size), dtype=torch.int8, device=device).view(dtype),
                   torch.zeros((blocks, 2, kv_heads), dtype=torch.float32, device=device), page_size, head_size)

    def append(self, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor, positions: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, rope_pairs: bool = False) -> Optional[torch.Tensor]:
        """Keys and values [rows, kv_heads, head_size] (float16 or bfloat16) to the slots of `slot_map` (a plan's), keys rotated by
        `rope` (rope_table) at `positions` if there is one, and queries `q` [rows, heads, head_size] with them: returns the rotated queries, in
        `q_out` (which may be q) or a new tensor.  rope_pairs: neighbours turn against each other, not halves.  Rows with a negative slot
        are passed over; their queries are left as q_out had them (a new tensor's are undefined)."""
        device, dtype, size, rows = self.pool.device, k.dtype, self.head_size, k.shape[0]
        if dtype not in _ACT:
            raise TypeError(f'keys have to be float16 or bfloat16: got {dtype}')
        rot = 0
        if rope is not None:
            if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or not rope.is_contiguous() or rope.device != device:
                raise ValueError(f'rope has to be contiguous float32 [positions, rot_dim / 2, 2] on {device}: got {rope.dtype} {tuple(rope.shape)} on {rope.device}')
            if positions is None:
                raise ValueError('rotation needs the positions')
            rot = 2 * rope.shape[1]
        if q is not None and not rot:
            raise ValueError('queries are only rotated here, and there is no rope table')
        kp, vp = _rows('k', k, rows, self.kv_heads, size, dtype, device), _rows('v', v, rows, self.kv_heads, size, dtype, device)
        qp = op = None
        q_heads, qs, os = 0, (0, 0), (0, 0)
        if q is not None:
            qp, q_heads, qs = _rows('q', q, rows, None, size, dtype, device), q.shape[1], _strides(q)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=dtype, device=device)
            op, os = _rows('q_out', q_out, rows, q_heads, size, dtype, device), _strides(q_out, True)
        ks, vs = _strides(k), _strides(v)
        p = _AppendParams(rows, self.kv_heads, q_heads, size, self.page_size, self.blocks, _ACT[dtype], self._type, rot, 1 if rope_pairs else 0,
                          rope.shape[0] if rot else 0, kp, vp, qp, op, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os[0], os[1],
                          _ints('slot_map', slot_map, rows, device), _ints('positions', positions, rows, device) if rot else None,
                          rope.data_ptr() if rot else None, self.pool.data_ptr(), self.scales.data_ptr())
        with _on(k) as stream:
            if _lib().tllm_paged_append(ctypes.addressof(p), stream):
                _raise('append')
        return q_out

    def attention(self, q: torch.Tensor, block_table: torch.Tensor, cu_tokens: torch.Tensor, kv_lens: torch.Tensor, max_new: int, max_kv: Optional[int] = None,
                  window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k) v of q [rows, heads, head_size] over the cached keys of each request, causal, the last `window` keys only if window > 0.
        Request b has the rows cu_tokens[b] .. cu_tokens[b + 1] and kv_lens[b] cached tokens, its rows the last of them.  `max_new`: no request has more
        rows; `max_kv`: the longest length to expect (default: what the tables hold), which only says how the work is split.  scale: 1 / sqrt(head_size)
        unless given.  Rows that belong to no request are left as `out` had them (a new tensor's are undefined)."""
        device, dtype, size, rows, n = self.pool.device, q.dtype, self.head_size, q.shape[0], kv_lens.numel()
        if dtype not in _ACT:
            raise TypeError(f'queries have to be float16 or bfloat16: got {dtype}')
        qp = _rows('q', q, rows, None, size, dtype, device)
        heads = q.shape[1]
        tp = _table(block_table, n, device)
        if out is None:
            out = torch.empty((rows, heads, size), dtype=dtype, device=device)
        op = _rows('out', out, rows, heads, size, dtype, device)
        wide = block_table.shape[1]
        qs, os = _strides(q), _strides(out, True)
        p = _AttentionParams(n, rows, heads, self.kv_heads, size, self.page_size, self.blocks, wide, _ACT[dtype], self._type, max_new,
                             wide * self.page_size if max_kv is None else max_kv, window, 1.0 / math.sqrt(size) if scale is None else scale, _table_stride(block_table),
                             qs[0], qs[1], os[0], os[1], qp, self.pool.data_ptr(), self.scales.data_ptr(), tp, _ints('cu_tokens', cu_tokens, n + 1, device),
                             _ints('kv_lens', kv_lens, None, device), op)
        at = ctypes.addressof(p)
        with _on(q) as stream:
            lib = _lib()
            need = lib.tllm_paged_attention_workspace(at)
            if need < 0:
                _raise('attention')
            work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            if lib.tllm_paged_attention(at, work.data_ptr() if need else None, stream):
                _raise('attention')
        return out
