"""Pages, an 8-bit cache and its attention for steps over packed batches (ctypes binding of include/tllm_serving_api.h).

Where KVCacheManager hands out block ids on the host, `DeviceBlockPool` keeps the free list, the tables and the lengths on the GPU: one
`plan` a step serves every layer, and nothing of it comes back to the host, so a step with it can be captured into a graph.  `PagedKV8Cache` is one
layer's cache: int8 or e4m3 elements (torch.int8, torch.float8_e4m3fn) under a scale for each page and head, filled by `append` and read by
`attention`.  Tensors are handed over as device pointers; calls run on torch's current stream of the tensors' device and check their
arguments (TypeError, ValueError; RuntimeError with the library's reason).  A failing call has launched nothing.  There are no gradients: these
operators serve."""
import ctypes
import struct
from typing import Optional

import torch

from ..plugin import capi

BF16 = 7
PAGE_SIZES, HEAD_SIZES = (16, 32, 64, 128), (64, 128, 256)
_ACT = {torch.float16: capi.HALF, torch.bfloat16: BF16}
_CACHE = {torch.int8: capi.INT8, torch.float8_e4m3fn: capi.FP8}

_INT = torch.int32
# the parameter structures of tllm_serving_api.h, in the platform's own layout
_PLAN, _APPEND, _ATTENTION = struct.Struct('@5iq11P'), struct.Struct('@11i4P8q5P'), struct.Struct('@13if5q7P')

_lib_ = None


def _lib():
    global _lib_
    if _lib_ is None:
        lib = capi.load_library()
        ptr = ctypes.c_void_p
        for name, args, result in (('tllm_paged_plan', [ptr, ptr], ctypes.c_int32), ('tllm_paged_append', [ptr, ptr], ctypes.c_int32),
                                   ('tllm_paged_attention', [ptr, ptr, ptr], ctypes.c_int32), ('tllm_paged_attention_workspace', [ptr], ctypes.c_int64)):
            f = getattr(lib, name)
            f.argtypes, f.restype = args, result
        _lib_ = lib
    return _lib_


def on_device(index: int, call, *args):
    """call(*args, stream) with device `index` as the current one and torch's current stream of it."""
    current = torch._C._cuda_getDevice()
    if current == index:
        return call(*args, torch._C._cuda_getCurrentRawStream(index))
    torch.cuda.set_device(index)
    try:
        return call(*args, torch._C._cuda_getCurrentRawStream(index))
    finally:
        torch.cuda.set_device(current)


def _no_number(e):
    raise ValueError(f'an argument is no number of its kind: {e}') from None


def _raise(name):
    raise RuntimeError(f'{name}: {capi.last_error()}')


def _got(t):
    return f'got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}'


def _ints(what, t, n, index):
    """The address of a contiguous int32 vector of n values on device `index`."""
    if t.dtype is _INT and t.shape == (n, ) and t.is_contiguous() and t.get_device() == index:
        return t.data_ptr()
    raise ValueError(f'{what} has to be a contiguous int32 vector of {n} values on GPU {index}: {_got(t)}')


def _table(t, rows, index):
    """Address, row stride and width of a table of `rows` rows or more."""
    if t.dtype is _INT and t.dim() == 2 and t.get_device() == index:
        (have, wide), (row, one) = t.shape, t.stride()
        if have >= rows and wide > 0 and (one == 1 or wide == 1):
            return t.data_ptr(), row if have > 1 else wide, wide
    raise ValueError(f'block_table has to be int32 [{rows} or more, blocks] with contiguous rows on GPU {index}: {_got(t)}')


def _rows(what, t, rows, heads, size, dtype, index, written=False):
    """Address, heads, row and head strides of [rows, heads, size] with a contiguous last dimension; views into packed projections are fine."""
    if t.dtype is dtype and t.dim() == 3 and t.get_device() == index:
        (n, h, d), (row, head, one) = t.shape, t.stride()
        if n == rows and d == size and one == 1 and (heads is None or h == heads):
            row, head = row if n > 1 else h * d, head if h > 1 else d  # of a dimension of one a stride says nothing
            if not written or (row >= d and head >= d):
                return t.data_ptr(), h, row, head
    raise ValueError(f'{what} has to be {dtype} [{rows}, {"heads" if heads is None else heads}, {size}] with a contiguous last dimension'
                     f'{", no two rows on one place," if written else ""} on GPU {index}: {_got(t)}')


class Fixed(object):
    """Attributes are set once: calls use the tensors that were checked, and do not check them again."""
    __slots__ = ()

    def __setattr__(self, name, value):
        if hasattr(self, name):
            raise AttributeError(f'{name} of a {type(self).__name__} stays what it is: make another one')
        object.__setattr__(self, name, value)


class StepPlan(Fixed):
    """What a step needs to know of its pages, in tensors that are written anew by every plan: cu_tokens [n_seqs + 1], slot_map and positions [n_rows]
    (-1 behind the last row), lens [n_seqs] and ring_state [2] behind the step, status [1] (0: fine; tllm_serving_api.h has the others).  The tensors
    stay the same ones for the plan's life."""
    __slots__ = ('n_seqs', 'n_rows', 'index', 'cu_tokens', 'slot_map', 'positions', 'status', 'lens', 'ring_state', '_at')

    def __init__(self, n_seqs: int, n_rows: int, device='cuda', lens: Optional[torch.Tensor] = None, ring_state: Optional[torch.Tensor] = None):
        new = lambda n: torch.empty(n, dtype=_INT, device=device)
        cu, slots, places, status = new(n_seqs + 1), new(n_rows), new(n_rows), new(1)
        index = cu.get_device()
        lens, ring_state = new(n_seqs) if lens is None else lens, new(2) if ring_state is None else ring_state
        at = (cu.data_ptr(), slots.data_ptr(), places.data_ptr(), _ints('lens', lens, n_seqs, index), _ints('ring_state', ring_state, 2, index), status.data_ptr())
        self.n_seqs, self.n_rows, self.index, self.cu_tokens, self.slot_map, self.positions, self.status, self.lens, self.ring_state, self._at = (
            n_seqs, n_rows, index, cu, slots, places, status, lens, ring_state, at)

    def __reduce_ex__(self, protocol):
        raise TypeError('a StepPlan is not copied: make another one')


def plan_step(lens: torch.Tensor, new_lens: torch.Tensor, ring: torch.Tensor, ring_state: torch.Tensor, block_table: torch.Tensor, page_size: int,
              n_rows: int, out: Optional[StepPlan] = None) -> StepPlan:
    """Pages for the step's tokens (tllm_paged_plan): lens and new_lens int32 [n], a negative new length ends a request.  `block_table` and `ring`
    are updated; the lengths and the ring's state behind the step are out.lens and out.ring_state, which may be `lens` and `ring_state`."""
    index, n = lens.get_device(), lens.numel()
    if index < 0:
        raise ValueError(f'the tensors have to be on a GPU: {_got(lens)}')
    if out is None:
        out = StepPlan(n, n_rows, lens.device)
    elif out.n_seqs != n or out.n_rows != n_rows or out.index != index:
        raise ValueError(f'out is a plan of {out.n_seqs} requests and {out.n_rows} rows on GPU {out.index}, the step has {n} and {n_rows} on GPU {index}')
    table, stride, wide = _table(block_table, n, index)
    blocks = ring.numel()
    try:
        p = _PLAN.pack(n, n_rows, page_size, blocks, wide, stride, _ints('lens', lens, n, index), _ints('new_lens', new_lens, n, index), _ints('ring', ring, blocks, index),
                       _ints('ring_state', ring_state, 2, index), table, *out._at)
    except struct.error as e:
        _no_number(e)
    if on_device(index, (_lib_ or _lib()).tllm_paged_plan, p):
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
        elif out.lens.data_ptr() != self.lens.data_ptr() or out.ring_state.data_ptr() != self.ring_state.data_ptr():
            raise ValueError('out has to be a plan over this pool: StepPlan(.., lens=pool.lens, ring_state=pool.ring_state)')
        return plan_step(self.lens, new_lens, self.ring, self.ring_state, self.block_table, self.page_size, n_rows, out)


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, factor: float = 1.0, device='cuda') -> torch.Tensor:
    """fp32 [positions, rot_dim / 2, 2]: cos and sin of position / factor * base^(-2 i / rot_dim), the angles formed in 64 bits."""
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / factor * base**(-2.0 * i / rot_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).to(device)


class PagedKV8Cache(Fixed):
    """One layer's cache: `pool` int8 or float8_e4m3fn [blocks, 2, kv_heads, page_size * head_size] (keys of a page and head [page_size, head_size],
    values [head_size, page_size]) and `scales` fp32 [blocks, 2, kv_heads].  The tensors are the caller's, the same ones for the cache's life;
    `PagedKV8Cache.empty` makes them."""

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
        self._index, self._at = pool.get_device(), (pool.data_ptr(), scales.data_ptr())

    def __reduce_ex__(self, protocol):  # copies have addresses of their own
        return type(self), (self.pool, self.scales, self.page_size, self.head_size)

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
        index, size, heads, dtype, rows = self._index, self.head_size, self.kv_heads, k.dtype, k.shape[0]
        act = _ACT.get(dtype)
        if act is None:
            raise TypeError(f'keys have to be float16 or bfloat16: got {dtype}')
        rot = places = angles = angle_rows = 0
        if rope is not None:
            if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or not rope.is_contiguous() or rope.get_device() != index:
                raise ValueError(f'rope has to be contiguous float32 [positions, rot_dim / 2, 2] on GPU {index}: {_got(rope)}')
            if positions is None:
                raise ValueError('rotation needs the positions')
            angle_rows, rot = rope.shape[0], 2 * rope.shape[1]
            places, angles = _ints('positions', positions, rows, index), rope.data_ptr()
        k_at, _, k_row, k_head = _rows('k', k, rows, heads, size, dtype, index)
        v_at, _, v_row, v_head = _rows('v', v, rows, heads, size, dtype, index)
        q_at = q_heads = q_row = q_head = o_at = o_row = o_head = 0
        if q is not None:
            if not rot:
                raise ValueError('queries are only rotated here, and there is no rope table')
            q_at, q_heads, q_row, q_head = _rows('q', q, rows, None, size, dtype, index)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            o_at, _, o_row, o_head = _rows('q_out', q_out, rows, q_heads, size, dtype, index, True)
        try:
            p = _APPEND.pack(rows, heads, q_heads, size, self.page_size, self.blocks, act, self._type, rot, 1 if rope_pairs else 0, angle_rows, k_at, v_at, q_at, o_at,
                             k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head, _ints('slot_map', slot_map, rows, index), places, angles, *self._at)
        except struct.error as e:
            _no_number(e)
        if on_device(index, (_lib_ or _lib()).tllm_paged_append, p):
            _raise('append')
        return q_out

    def attention(self, q: torch.Tensor, block_table: torch.Tensor, cu_tokens: torch.Tensor, kv_lens: torch.Tensor, max_new: int, max_kv: Optional[int] = None,
                  window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale q k) v of q [rows, heads, head_size] over the cached keys of each request, causal, the last `window` keys only if window > 0.
        Request b has the rows cu_tokens[b] .. cu_tokens[b + 1] and kv_lens[b] cached tokens, its rows the last of them.  `max_new`: no request has more
        rows; `max_kv`: the longest length to expect (default: what the tables hold), which only says how the work is split.  scale: 1 / sqrt(head_size)
        unless given; `out` may be q.  Rows that belong to no request are left as `out` had them (a new tensor's are undefined)."""
        index, size, dtype, rows, n = self._index, self.head_size, q.dtype, q.shape[0], kv_lens.numel()
        act = _ACT.get(dtype)
        if act is None:
            raise TypeError(f'queries have to be float16 or bfloat16: got {dtype}')
        q_at, heads, q_row, q_head = _rows('q', q, rows, None, size, dtype, index)
        table, stride, wide = _table(block_table, n, index)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        o_at, _, o_row, o_head = _rows('out', out, rows, heads, size, dtype, index, True)
        try:
            p = _ATTENTION.pack(n, rows, heads, self.kv_heads, size, self.page_size, self.blocks, wide, act, self._type, max_new,
                                wide * self.page_size if max_kv is None else max_kv, window, size**-0.5 if scale is None else scale, stride, q_row, q_head, o_row, o_head,
                                q_at, *self._at, table, _ints('cu_tokens', cu_tokens, n + 1, index), _ints('kv_lens', kv_lens, n, index), o_at)
        except struct.error as e:
            _no_number(e)
        if on_device(index, self._attend, p):
            _raise('attention')
        return out

    def _attend(self, p, stream):
        lib = _lib_ or _lib()
        need = lib.tllm_paged_attention_workspace(p)
        if need <= 0:  # none, or refused: the call says why
            return lib.tllm_paged_attention(p, None, stream)
        workspace = torch.empty(need, dtype=torch.uint8, device=self.pool.device)  # held over the call: another thread could be given it between the launches
        return lib.tllm_paged_attention(p, workspace.data_ptr(), stream)
