"""Linear layers with 4-bit weights and a scale for each group of a row (ctypes binding of tllm_group_matmul, include/tllm_serving_api.h).

Next to WeightOnlyQuantMatmul, whose 4-bit weights have one scale for a whole output channel.  y = x W^T, W[n, k] = q[n, k] s[n, k / group].  There are no
gradients: the product serves."""
import ctypes
import struct
from typing import Optional, Tuple

import torch

from ..plugin import capi
from ..runtime.paged_kv8 import Fixed, on_device

GROUPS = (32, 64, 128)
_ACT = {torch.float16: capi.HALF, torch.bfloat16: 7}
_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # element of a word's eight that nibble i holds

_PARAMS = struct.Struct('@5i2q4P')  # tllm_group_matmul_params_t

_matmul = None


def _entry():
    global _matmul
    if _matmul is None:
        f = capi.load_library().tllm_group_matmul
        f.argtypes, f.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int32
        _matmul = f
    return _matmul


def _checked(n: int, k: int, group: int):
    if group not in GROUPS:
        raise ValueError(f'group is one of {GROUPS}: got {group}')
    if n < 1 or k < 32 or k % 32:
        raise ValueError(f'weights are [n, k] with k a multiple of 32: got [{n}, {k}]')


def quantize(weight: torch.Tensor, group: int, dtype=torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """weight [n, k] -> (q int8 [n, k] in -8 .. 7, scales `dtype` [n, ceil(k / group)]): the scale is the group's largest magnitude / 7 rounded to
    `dtype` (1 for a group of zeros, and for one whose scale would round to 0), q the nearest even of weight / scale."""
    n, k = weight.shape
    _checked(n, k, group)
    count = -(-k // group)
    w = torch.zeros((n, count * group), dtype=torch.float32, device=weight.device)
    w[:, :k] = weight.detach()
    w = w.view(n, count, group)
    scales = (w.abs().amax(-1) / 7).to(dtype)
    if not bool(torch.isfinite(scales).all()):
        raise ValueError(f'the weights have a group whose scale is not finite in {dtype}')
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    q = torch.round(w / scales.float()[..., None]).clamp_(-8, 7).to(torch.int8)
    return q.view(n, -1)[:, :k].contiguous(), scales


def pack(q: torch.Tensor, scales: torch.Tensor, group: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """q int8 [n, k] in -8 .. 7 and scales [n, ceil(k / group)] -> what the kernel reads (the layout is in tllm_serving_api.h), on the same device."""
    n, k = q.shape
    _checked(n, k, group)
    if q.dtype is not torch.int8 or scales.dtype not in _ACT or tuple(scales.shape) != (n, -(-k // group)) or scales.device != q.device:
        raise ValueError(f'q has to be int8 [n, k] and the scales float16 or bfloat16 [n, {-(-k // group)}] on one device: got {q.dtype} {tuple(q.shape)}, '
                         f'{scales.dtype} {tuple(scales.shape)}')
    if int(q.min()) < -8 or int(q.max()) > 7:
        raise ValueError('q has values outside -8 .. 7')
    scales = scales.detach()
    tiles, steps = -(-n // 16), -(-k // 128)
    u = torch.full((16 * tiles, 128 * steps), 8, dtype=torch.uint8, device=q.device)
    u[:n, :k] = (q + 8).to(torch.uint8)
    u = u.view(tiles, 16, steps, 4, 4, 8)[..., _ORDER]  # [tile, r, k tile, j, g, nibble]
    u = (u[..., 0::2] | (u[..., 1::2] << 4)).permute(0, 2, 4, 1, 3, 5)  # [tile, k tile, g, r, j, byte]
    s = torch.zeros((scales.shape[1], 16 * tiles), dtype=scales.dtype, device=q.device)
    s[:, :n] = scales.t()
    return u.reshape(tiles, steps, 64, 16).contiguous(), s


def _restored(cls, *held):
    layer = cls.__new__(cls)
    layer._hold(*held)
    return layer


class GroupQuantMatmul(Fixed):
    """y = x W^T with W packed once: q int8 [n, k] in -8 .. 7, scales float16 or bfloat16 [n, ceil(k / group)], which is the type of x and y too."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, group: int):
        self._hold(*q.shape, group, *pack(q, scales, group))

    def _hold(self, n, k, group, packed, scales):
        self.n, self.k, self.group, self.dtype, self.packed, self.scales = n, k, group, scales.dtype, packed, scales
        if self.packed.device.type != 'cuda':
            raise ValueError(f'the weights have to be on a GPU: got {self.packed.device}')
        self._index, self._act, self._at = self.packed.get_device(), _ACT[self.dtype], (self.packed.data_ptr(), self.scales.data_ptr())

    def __reduce_ex__(self, protocol):  # copies have addresses of their own
        return _restored, (type(self), self.n, self.k, self.group, self.packed, self.scales)

    @classmethod
    def from_float(cls, weight: torch.Tensor, group: int, dtype=torch.float16) -> 'GroupQuantMatmul':
        return cls(*quantize(weight, group, dtype), group)

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [.., k] -> [.., n]; a two-dimensional x may have strided rows.  `out` [rows, n] takes the result if given; it does not overlap x."""
        index, n, k = self._index, self.n, self.k
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        (rows, wide), (row, one) = x2.shape, x2.stride()
        if x.dtype is not self.dtype or wide != k or one != 1 or x.get_device() != index:
            raise ValueError(f'x has to be {self.dtype} [.., {k}] with contiguous rows on GPU {index}: got {x.dtype} {tuple(x.shape)} with strides {x.stride()} on {x.device}')
        if out is None:
            y, y_row = torch.empty((rows, n), dtype=self.dtype, device=x.device), n
        else:
            y, y_row = out, out.stride(0) if rows > 1 else n
            if y.dtype is not self.dtype or tuple(y.shape) != (rows, n) or (y.stride(1) != 1 and n > 1) or y.get_device() != index:
                raise ValueError(f'out has to be {self.dtype} [{rows}, {n}] with contiguous rows on GPU {index}: got {y.dtype} {tuple(y.shape)} with strides {y.stride()} on {y.device}')
        p = _PARAMS.pack(rows, n, k, self.group, self._act, row if rows > 1 else k, y_row, x2.data_ptr(), *self._at, y.data_ptr())
        if on_device(index, _matmul or _entry(), p):
            raise RuntimeError(f'GroupQuantMatmul: {capi.last_error()}')
        return y if out is not None or x.dim() == 2 else y.view(*x.shape[:-1], n)
