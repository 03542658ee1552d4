"""4-bit microscaled matrices without a GPU: the storage form, its import and
export, and every refusal (each fires before any launch)."""
import ctypes

import numpy as np
import pytest
import torch

import _mx4
from custom_matmul_kernels_amd import MX4BMMCUDA, MX4Tensor, _lib, quantize_mx4


def blocks(l, rows, k, seed=0):
    gen = torch.Generator().manual_seed(seed)
    codes, scales = _mx4.encode(torch.randn(l, rows, k, generator=gen))
    return torch.from_numpy(_mx4.packed(codes)), torch.from_numpy(scales)


def test_oracle_rounds_ties_to_even_and_saturates():
    q = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.5, 6.0, 7.9, 0.2501, -0.75, -2.5, 0.0, 4.0])
    want = np.array([0, 1, 1, 2, 2, 4, 4, 6, 6, 6, 0.5, -1, -2, 0, 4])
    x = np.concatenate([q, np.zeros(32 - len(q))])           # largest 7.9: scale 1
    codes, scales = _mx4.encode(x)
    assert scales[0] == 127
    assert np.array_equal(_mx4.decode(codes, scales)[:len(q)], want)


@pytest.mark.parametrize("k", [1, 31, 32, 33, 96, 128, 129, 200, 256])
@pytest.mark.parametrize("rows", [1, 3, 17])
def test_blocks_survive_the_storage_form(rows, k):
    codes, scales = blocks(2, rows, k)
    t = MX4Tensor.from_blocks(codes, scales, k)
    assert t.shape == (2, rows, k) and t.rows == rows
    assert tuple(t.codes.shape) == (2, -(-k // 128), rows, 64)
    back = t.blocks()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)
    # element (l, r, i) sits at slab i // 128, byte (i % 128) // 2, low half first
    for i in {0, k // 2, k - 1}:
        byte = t.codes[1, i // 128, rows - 1, i % 128 // 2].item()
        assert byte >> (4 * (i % 2)) & 15 == codes[1, rows - 1, i // 2].item() >> (4 * (i % 2)) & 15
        assert t.scales[1, i // 128, rows - 1, i % 128 // 32] == scales[1, rows - 1, i // 32]


def test_codes_beyond_k_are_cleared_on_import():
    codes = torch.full((1, 2, 32), 0x55, dtype=torch.uint8)
    scales = torch.full((1, 2, 2), 127, dtype=torch.uint8)
    t = MX4Tensor.from_blocks(codes, scales, 35)
    assert (t.codes[0, 0, :, :17] == 0x55).all() and (t.codes[0, 0, :, 17] == 5).all()
    assert (t.codes[0, 0, :, 18:] == 0).all() and (t.scales[0, 0, :, 2:] == 0).all()


def test_transpose_and_two_dimensions():
    codes, scales = blocks(1, 5, 40)
    t = MX4Tensor.from_blocks(codes[0], scales[0], 40)
    assert t.shape == (5, 40) and t.dim() == 2
    u = t.transpose(0, 1)
    assert u.shape == (40, 5) and u.k_axis == -2 and u.codes is t.codes
    assert u.transpose().shape == (5, 40)
    with pytest.raises(AssertionError):
        MX4Tensor.from_blocks(codes, scales, 40).transpose(0, 1)


def test_wrong_storage_is_refused():
    codes, scales = blocks(1, 5, 40)
    t = MX4Tensor.from_blocks(codes, scales, 40)
    with pytest.raises(TypeError):
        MX4Tensor(t.codes.int(), t.scales, 40)
    with pytest.raises(TypeError):
        MX4Tensor.from_blocks(codes.int(), scales, 40)
    for bad in (lambda: MX4Tensor(t.codes, t.scales, 129), lambda: MX4Tensor(t.codes, t.scales[:, :, :4], 40),
                lambda: MX4Tensor(t.codes, t.scales, 40, k_axis=0),
                lambda: MX4Tensor(t.codes.transpose(1, 2), t.scales, 40),
                lambda: MX4Tensor.from_blocks(codes, scales, 70),
                lambda: MX4Tensor.from_blocks(codes, scales[:, :, :1], 40)):
        with pytest.raises(AssertionError):
            bad()


def test_refusals_of_the_python_entry_points():
    codes, scales = blocks(2, 5, 40)
    A = MX4Tensor.from_blocks(codes, scales, 40)                       # [2, 5, 40]
    B = A.transpose()                                                  # [2, 40, 5]
    product = MX4BMMCUDA()
    with pytest.raises(TypeError):
        MX4BMMCUDA(out_dtype=torch.float64)
    with pytest.raises(TypeError):
        quantize_mx4(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(ValueError):
        quantize_mx4(torch.zeros(3))
    with pytest.raises(ValueError):
        quantize_mx4(torch.zeros(3, 3, 3, 3))
    for dim in (0, -3, 3):
        with pytest.raises(AssertionError):
            quantize_mx4(torch.zeros(2, 3, 4), dim=dim)
    with pytest.raises(AssertionError):
        quantize_mx4(torch.zeros(2, 3, 4))                             # not on a device
    with pytest.raises(AssertionError):
        A.dequantize()
    with pytest.raises(TypeError):
        A.dequantize(torch.int32)
    with pytest.raises(AssertionError):
        product(A, B)                                                  # not on a device
    with pytest.raises(AssertionError):
        product(A, A)                                                  # blocks of B do not run along k
    with pytest.raises(AssertionError):
        product(B, B)
    with pytest.raises(AssertionError):
        product(torch.zeros(2, 5, 41), B)                              # contraction mismatch
    with pytest.raises(AssertionError):
        product(torch.zeros(3, 5, 40), B)                              # batch mismatch
    with pytest.raises(AssertionError):
        product(torch.zeros(5, 40), B)                                 # 2d against 3d
    with pytest.raises(TypeError):
        product(torch.zeros(2, 5, 40, dtype=torch.float64), B)
    with pytest.raises(RuntimeError, match="backward"):
        product(torch.zeros(2, 5, 40, requires_grad=True), B)
    with pytest.raises(AssertionError):                                # passes the gradient check without grad
        with torch.no_grad():
            product(torch.zeros(2, 5, 40, requires_grad=True), B)


def test_refusals_of_the_c_entry_points():
    lib = _lib.load()
    ok, odd = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1002)          # never dereferenced
    bad = _lib.ERR_INVALID_ARG
    assert lib.cmk_mx4_quantize(ok, 3, ok, ok, 1, 1, 1, 1, 1, 1, None) == bad
    assert lib.cmk_mx4_quantize(ok, 0, ok, ok, 1, -1, 1, 1, 1, 1, None) == bad
    assert lib.cmk_mx4_quantize(None, 0, ok, ok, 1, 1, 1, 1, 1, 1, None) == bad
    assert lib.cmk_mx4_quantize(ok, 0, odd, ok, 1, 1, 1, 1, 1, 1, None) == bad
    assert b"alignment" in lib.cmk_last_error()
    assert lib.cmk_mx4_quantize(ok, 0, ok, odd, 1, 1, 1, 1, 1, 1, None) == bad
    assert lib.cmk_mx4_dequantize(ok, ok, ok, -1, 1, 1, 1, 0, None) == bad
    assert lib.cmk_mx4_dequantize(ok, ok, None, 0, 1, 1, 1, 0, None) == bad
    assert lib.cmk_mx4_dequantize(odd, ok, ok, 0, 1, 1, 1, 0, None) == bad
    def four(data=ok, scales=ok):
        return _lib.Mx4Operand(data, scales, _lib.MX4)

    def floats(data=ok, dtype=_lib.F32, sk=1):
        return _lib.Mx4Operand(data, None, dtype, 0, 1, 1, sk)

    def bmm(a, b, c=ok, dtype=0, l=1, m=1, n=1, k=1, ws=None, nbytes=0):
        return lib.cmk_mx4_bmm(a, b, c, dtype, l, m, n, k, ws, nbytes, None)

    def need(a, b, l, m, n, k):
        return lib.cmk_mx4_workspace_bytes(a, b, l, m, n, k)

    assert bmm(None, four()) == bad
    assert bmm(four(), four(), dtype=7) == bad
    assert bmm(four(), four(), dtype=_lib.MX4) == bad
    assert bmm(floats(dtype=9), four()) == bad
    assert bmm(four(), four(), n=-1) == bad
    assert bmm(four(), four(), c=None) == bad
    assert bmm(four(), four(), m=(1 << 30) + 1) == bmm(four(), four(), n=(1 << 30) + 1) == _lib.ERR_UNSUPPORTED
    assert bmm(four(), four(data=None)) == bad
    assert bmm(four(scales=None), four()) == bad
    assert bmm(four(), four(data=odd)) == bad
    assert bmm(four(scales=odd), four()) == bad
    assert bmm(floats(data=None), four()) == bad
    # few tiles and a long contraction: a workspace, and a refusal without it
    size = need(four(), four(), 1, 128, 128, 16384)
    assert size > 0 and size % (128 * 128 * 4) == 0
    assert need(four(), four(), 1, 8192, 8192, 8192) == need(four(), four(), 1, 1, 64, 65536) == 0
    fault = _lib.ERR_WORKSPACE
    assert bmm(four(), four(), m=128, n=128, k=16384) == fault
    assert bmm(four(), four(), m=128, n=128, k=16384, ws=ok, nbytes=size - 1) == fault
    assert bmm(four(), four(), m=128, n=128, k=16384, ws=ctypes.c_void_p(0x1010), nbytes=size) == fault
    # operands that are quantised in the call need room for their 4-bit form, a left one of few rows does not
    assert need(floats(), four(), 1, 4, 512, 1000) == 0
    assert need(floats(sk=7), four(), 1, 4, 512, 1000) >= 8 * 4 * 68
    assert need(floats(), floats(), 2, 100, 512, 1000) >= 2 * 8 * (100 + 512) * 68
    assert bmm(four(), floats()) == fault and bmm(floats(), floats()) == fault
    assert need(None, four(), 1, 1, 1, 1) == need(four(), four(), 1, 0, 1, 1) == need(floats(dtype=9), four(), 1, 1, 1, 1) == 0
    # nothing to do is no error
    assert lib.cmk_mx4_quantize(None, 0, None, None, 1, 0, 5, 1, 1, 1, None) == 0
    assert lib.cmk_mx4_dequantize(None, None, None, 0, 0, 5, 5, 0, None) == 0
    assert bmm(four(None, None), four(None, None), c=None, m=0, n=5, k=5) == 0


def test_operand_layout_matches_header():
    assert ctypes.sizeof(_lib.Mx4Operand) == 48
    assert _lib.Mx4Operand.stride_l.offset == 24


def test_more_than_a_launch_holds_is_refused():
    """2^24 work-groups of 256 threads are 2^32 threads, which wrap round in a launch."""
    lib = _lib.load()
    ok = ctypes.c_void_p(0x1000)          # never dereferenced
    four = _lib.Mx4Operand(ok, ok, _lib.MX4)
    large = 1 << 26                       # matrices of one row: a wave each
    assert lib.cmk_mx4_quantize(ok, 0, ok, ok, large, 1, 1, 1, 1, 1, None) == _lib.ERR_UNSUPPORTED
    assert b"more than a launch holds" in lib.cmk_last_error()
    assert lib.cmk_mx4_quantize(ok, 0, ok, ok, large, 1, 4, 1, 1, 2, None) == _lib.ERR_UNSUPPORTED
    for rows_innermost in (0, 1):
        assert lib.cmk_mx4_dequantize(ok, ok, ok, 0, large, 1, 1, rows_innermost, None) == _lib.ERR_UNSUPPORTED
    for m, n in [(1, 1), (64, 64)]:       # a work-group each
        assert lib.cmk_mx4_bmm(four, four, ok, 0, 1 << 24, m, n, 32, None, 0, None) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("large", [2 ** 31, 2 ** 32, 2 ** 32 + 128])
def test_extents_beyond_a_c_int_are_refused(large):
    """They would reach the library cut to 32 bits; meta tensors hold no elements."""
    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")
    for shape in ((1, large), (large, 1), (large, 1, 1), (2, 3, large)):
        for dim in (-1, -2):
            with pytest.raises(ValueError, match="2\\^31"):
                quantize_mx4(meta(*shape), dim=dim)
    product = MX4BMMCUDA()
    for a, b in (((1, large), (large, 1)), ((large, 4), (4, 1)), ((1, 4), (4, large)), ((large, 1, 1), (large, 1, 1))):
        with pytest.raises(ValueError, match="2\\^31"):
            product(meta(*a), meta(*b))
    slabs = -(-large // 128)
    u8 = dict(dtype=torch.uint8)
    with pytest.raises(ValueError, match="2\\^31"):
        MX4Tensor(meta(1, slabs, 1, 64, **u8), meta(1, slabs, 1, 4, **u8), large)
    with pytest.raises(ValueError, match="2\\^31"):
        MX4Tensor(meta(1, 1, large, 64, **u8), meta(1, 1, large, 4, **u8), 5)
    with pytest.raises(ValueError, match="2\\^31"):
        MX4Tensor.from_blocks(meta(1, -(-large // 32) * 16, **u8), meta(1, -(-large // 32), **u8), large)


def test_few_rows_take_tiles_where_a_launch_would_wrap_round():
    """64 columns a work-group of 512 threads: 2^23 of them are 2^32 threads.  The kernel
    for few rows quantises a float left operand by itself and needs no room for it."""
    lib = _lib.load()
    ok = ctypes.c_void_p(0x1000)          # never dereferenced
    left, right = _lib.Mx4Operand(ok, None, _lib.F32, 0, 0, 128, 1), _lib.Mx4Operand(ok, ok, _lib.MX4)
    for m in (1, 8):
        assert lib.cmk_mx4_workspace_bytes(left, right, 1, m, (1 << 29) - 64, 128) == 0
        assert lib.cmk_mx4_workspace_bytes(left, right, 1, m, (1 << 29) - 63, 128) > 0
        assert lib.cmk_mx4_workspace_bytes(left, right, 1, m, 1 << 29, 128) > 0


def test_tangents_of_forward_mode_are_refused():
    """A dual tensor does not require grad, and its tangent must not be dropped in silence."""
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.randn(4, 40), torch.randn(40, 5)
    product = MX4BMMCUDA()
    with forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        assert not dx.requires_grad
        for args in ((dx, w), (x, dw)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                product(*args)
        with pytest.raises(AssertionError):                            # not on a device: no tangent, no refusal
            product(x, w)
        with pytest.raises(AssertionError):
            product(forward_ad.unpack_dual(dx).primal, w)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: product(v, w), (x,), (x,))


def test_quantisation_refuses_what_has_a_derivative():
    """(The check of the device comes first without a GPU.)"""
    import torch.autograd.forward_ad as forward_ad
    from custom_matmul_kernels_amd import _common
    x = torch.randn(4, 40)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            _common.refuse_grad(dual)
        _common.refuse_grad(x)
    _common.refuse_grad(x)
    with pytest.raises(RuntimeError, match="backward"):
        _common.refuse_grad(x.requires_grad_())
