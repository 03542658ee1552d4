"""Matrices in 4-bit microscaled floating point: quantisation, its inverse and
the batched product on the matrix pipe's scaled instructions.  No counterpart in
the reference, whose products are fp32; the class stands beside BMMCUDA."""
import torch
from torch.autograd import forward_ad

from . import _common, _lib

BLOCK = 32        # elements along k that share a scale
SLAB = 128        # elements of k that lie together in storage


class MX4Tensor:
    """One [r, c] or a batch of [l, r, c] matrices in 4 bits, made by
    ``quantize_mx4`` or ``MX4Tensor.from_blocks``.

    Blocks of 32 elements along one of the last two axes (the contraction axis
    of a product, `k_axis`, -1 or -2) share a power-of-two scale.  With the other
    axis called rows:
        codes  uint8 [l, ceil(k/128), rows, 64]: two elements a byte, the even
               index in the low half; bit 3 is the sign, the rest indexes
               0, .5, 1, 1.5, 2, 3, 4, 6
        scales uint8 [l, ceil(k/128), rows, 4]: byte s stands for 2^(s-127), 255
               for NaN
    Elements beyond k are zero codes.  ``transpose`` swaps the matrix axes and
    shares the storage."""

    def __init__(self, codes, scales, k, k_axis=-1, two_dimensional=False):
        slabs = -(-k // SLAB)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be torch.uint8")
        assert k_axis in (-1, -2)
        _common.check_extents(*codes.shape, k)
        assert codes.dim() == 4 and codes.shape[1] == slabs and codes.shape[3] == SLAB // 2
        assert tuple(scales.shape) == tuple(codes.shape[:3]) + (SLAB // BLOCK,)
        assert codes.device == scales.device
        assert codes.is_contiguous() and scales.is_contiguous()
        assert codes.data_ptr() % 16 == 0 and scales.data_ptr() % 4 == 0
        assert not two_dimensional or codes.shape[0] == 1
        self._set((codes, scales), codes.shape[0], codes.shape[2], k, k_axis, two_dimensional)

    def _set(self, storage, batch, rows, k, k_axis, two_dimensional):
        # storage: (codes, scales), or one buffer that holds the codes and behind
        # them the scales (one allocation less per call of quantize_mx4)
        self._storage = storage
        self.batch, self.rows, self.k, self.k_axis = batch, rows, k, k_axis
        self.two_dimensional = two_dimensional
        self.device = storage[0].device if type(storage) is tuple else storage.device
        matrix = (rows, k) if k_axis == -1 else (k, rows)
        self.shape = matrix if two_dimensional else (batch,) + matrix

    @classmethod
    def _wrap(cls, *args):
        t = object.__new__(cls)
        t._set(*args)
        return t

    def _blocks4(self):
        return self.batch * -(-self.k // SLAB) * self.rows

    def _pointers(self):
        if type(self._storage) is tuple:
            return self._storage[0].data_ptr(), self._storage[1].data_ptr()
        p = self._storage.data_ptr()
        return p, p + self._blocks4() * (SLAB // 2)

    def _views(self):
        if type(self._storage) is not tuple:
            head, n = (self.batch, -(-self.k // SLAB), self.rows), self._blocks4() * (SLAB // 2)
            self._storage = (self._storage[:n].view(head + (SLAB // 2,)),
                             self._storage[n:].view(head + (SLAB // BLOCK,)))
        return self._storage

    @property
    def codes(self):
        return self._views()[0]

    @property
    def scales(self):
        return self._views()[1]

    def dim(self):
        return 2 if self.two_dimensional else 3

    def transpose(self, dim0=-2, dim1=-1):
        n = self.dim()
        assert {dim0 % n, dim1 % n} == {n - 2, n - 1}, "only the two matrix axes can be swapped"
        return MX4Tensor._wrap(self._storage, self.batch, self.rows, self.k, -3 - self.k_axis, self.two_dimensional)

    def to(self, device):
        return MX4Tensor(self.codes.to(device), self.scales.to(device), self.k, self.k_axis, self.two_dimensional)

    def dequantize(self, dtype=torch.float32):
        """The values as a dense tensor of `shape`.  In float32 and bfloat16 they
        are exact; in float16 they are rounded where its range ends."""
        code = _common.float_type(dtype, "dtype")
        assert self.device.type == "cuda"
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        if out.numel():
            codes, scales = self._pointers()
            _common.call(_lib.load().cmk_mx4_dequantize, self.device, codes, scales, out.data_ptr(), code,
                         self.batch, self.rows, self.k, 1 if self.k_axis == -2 else 0)
        return out

    @classmethod
    def from_blocks(cls, codes, scales, k, k_axis=-1):
        """From row-major blocks, as checkpoints hold them: codes uint8
        [(l,) rows, ceil(k/32)*16], scales uint8 [(l,) rows, ceil(k/32)].  Codes
        beyond k have to be zero and are cleared here."""
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be torch.uint8")
        assert codes.dim() == scales.dim() and codes.dim() in (2, 3)
        two_dimensional = codes.dim() == 2
        if two_dimensional:
            codes, scales = codes[None], scales[None]
        blocks = -(-k // BLOCK)
        l, rows, _ = codes.shape
        _common.check_extents(l, rows, k)
        assert tuple(codes.shape) == (l, rows, blocks * BLOCK // 2)
        assert tuple(scales.shape) == (l, rows, blocks)
        slabs = -(-k // SLAB)
        c = torch.zeros(l, rows, slabs * SLAB // 2, dtype=torch.uint8, device=codes.device)
        c[:, :, :k // 2] = codes[:, :, :k // 2]
        if k % 2:
            c[:, :, k // 2] = codes[:, :, k // 2] & 15
        s = torch.zeros(l, rows, slabs * SLAB // BLOCK, dtype=torch.uint8, device=codes.device)
        s[:, :, :blocks] = scales
        c = c.view(l, rows, slabs, SLAB // 2).transpose(1, 2).contiguous()
        s = s.view(l, rows, slabs, SLAB // BLOCK).transpose(1, 2).contiguous()
        return cls(c, s, k, k_axis, two_dimensional)

    def blocks(self):
        """(codes, scales) in the row-major form that ``from_blocks`` takes."""
        l, slabs, rows, _ = self.codes.shape
        n = -(-self.k // BLOCK)
        c = self.codes.transpose(1, 2).reshape(l, rows, slabs * SLAB // 2)[:, :, :n * BLOCK // 2].contiguous()
        s = self.scales.transpose(1, 2).reshape(l, rows, slabs * SLAB // BLOCK)[:, :, :n].contiguous()
        return (c[0], s[0]) if self.two_dimensional else (c, s)


def quantize_mx4(T, dim=-1):
    """The 4-bit form of a device tensor [r, c] or [l, r, c] of float32, bfloat16
    or float16 with any strides; `dim`, the axis along which 32 elements share a
    scale, is one of the last two: -1 for the left operand of a product, -2 for
    the right one."""
    dtype = _common.float_type(T.dtype, "the tensor")
    if T.is_neg():
        T = _common.with_own_sign(T)
    shape, stride, device = T.shape, T.stride(), T.device
    n = len(shape)
    if n not in (2, 3):
        raise ValueError("the tensor needs to be 2d or 3d")
    k_axis = dim if dim < 0 else dim - n
    assert k_axis == -1 or k_axis == -2, "dim must be one of the two matrix axes"
    l = 1 if n == 2 else shape[0]
    rows, k = shape[-3 - k_axis], shape[k_axis]
    if l | rows | k > _common.MAX_EXTENT:
        _common.check_extents(l, rows, k)
    assert device.type == "cuda"
    if T.requires_grad or forward_ad._current_level >= 0:
        _common.refuse_grad(T)
    units = l * -(-k // SLAB) * rows
    storage = torch.empty(units * (SLAB // 2 + SLAB // BLOCK), dtype=torch.uint8, device=device)
    if units:
        p = storage.data_ptr()
        _common.call(_lib.load().cmk_mx4_quantize, device, T.data_ptr(), dtype, p, p + units * (SLAB // 2), l, rows, k,
                     0 if n == 2 else stride[0], stride[-3 - k_axis], stride[k_axis])
    return MX4Tensor._wrap(storage, l, rows, k, k_axis, n == 2)


class MX4BMMCUDA:
    """Batched product of operands in 4 bits: ``MX4BMMCUDA(out_dtype)(A, B)`` is
    C = A @ B with A [l, m, k] or [m, k], B [l, k, n] or [k, n] and C in
    `out_dtype` (float32, bfloat16 or float16).

    An operand is an MX4Tensor whose blocks run along k (A: ``dim=-1``, B:
    ``dim=-2``) or a float tensor, which is quantised in the call.  Sums are held
    in fp32 and rounded once.  There is no backward pass and no forward-mode
    derivative: operands that ask for one are refused."""

    def __init__(self, out_dtype=torch.float32):
        self._out = _common.float_type(out_dtype, "out_dtype")
        self.out_dtype = out_dtype
        self._lib = _lib.load()

    @staticmethod
    def _operand(T, k_axis, name):
        """The operand [l, rows, k] with k at `k_axis`, to be kept until the launch, and the
        library's description of it."""
        if isinstance(T, MX4Tensor):
            assert T.k_axis == k_axis, "the blocks of %s must run along k" % name
            return T, _lib.Mx4Operand(*T._pointers(), _lib.MX4)
        dtype = _common.float_type(T.dtype, name)
        if T.requires_grad or forward_ad._current_level >= 0:
            _common.refuse_grad(T)
        if T.is_neg():
            T = _common.with_own_sign(T)
        stride = T.stride()
        return T, _lib.Mx4Operand(T.data_ptr(), None, dtype, 0, stride[0] if len(stride) == 3 else 0,
                               stride[-3 - k_axis], stride[k_axis])

    def __call__(self, A, B):
        sa, sb, device = A.shape, B.shape, A.device
        n = len(sa)
        assert len(sb) == n
        if n not in (2, 3):
            raise ValueError("A and B need to be 2d or 3d")
        A, a = self._operand(A, -1, "A")
        B, b = self._operand(B, -2, "B")
        m, k = sa[-2:]
        c = sb[-1]
        l = 1 if n == 2 else sa[0]
        assert sb[-2] == k
        assert n == 2 or sb[0] == l
        if l | m | c | k > _common.MAX_EXTENT:
            _common.check_extents(l, m, c, k)
        assert device.type == "cuda"
        assert device == B.device
        C = torch.empty((m, c) if n == 2 else (l, m, c), dtype=self.out_dtype, device=device)
        if l and m and c:
            _common.call_with_workspace(self._lib.cmk_mx4_workspace_bytes, self._lib.cmk_mx4_bmm, device, (a, b, l, m, c, k),
                                        (a, b, C.data_ptr(), self._out, l, m, c, k))
        return C
