"""Mixture-of-experts layer without a GPU: every refusal fires before any launch."""
import ctypes

import pytest
import torch

import _mx4
from custom_matmul_kernels_amd import MoECUDA, MX4Tensor, _lib


def operands(t=3, h=64, i=32, e=4, dtype=torch.bfloat16):
    return (torch.zeros(t, h, dtype=dtype), torch.zeros(e, h, dtype=dtype),
            torch.zeros(e, 2 * i, h, dtype=dtype), torch.zeros(e, h, i, dtype=dtype))


def test_constructor_refusals():
    with pytest.raises(ValueError):
        MoECUDA(activation="relu")
    with pytest.raises(AssertionError):
        MoECUDA(k=0)
    with pytest.raises(AssertionError):
        MoECUDA(renormalize=1)


def test_call_refusals():
    layer = MoECUDA(k=2)
    x, r, g, d = operands()
    bad_type = [(x.float(), r, g, d), (x, r.half(), g, d), (x, r.double(), g, d), (x, r, g.half(), d), (x, r, g, d.float())]
    for args in bad_type:
        with pytest.raises(TypeError):
            layer(*args)
    for args in ((x[0], r, g, d), (x, r[0], g, d), (x, r, g[0], d), (x, r, g, d[0]),
                 (x, r, g.transpose(1, 2).contiguous().transpose(1, 2), d),
                 (x, r, g, d.transpose(1, 2).contiguous().transpose(1, 2)),
                 (x, r, g[:, :, :1].expand(4, 64, 64), d)):
        with pytest.raises(ValueError):
            layer(*args)
    for args in ((x[:, :63], r, g, d), (x, r[:3], g, d), (x, r, g[:, :63], d), (x, r, g[:3], d), (x, r, g, d[:, :63]),
                 (x, r, g, d[:, :, :31]), (x, r, g, d)):
        with pytest.raises(AssertionError):             # the last one: not on a device
            layer(*args)
    with pytest.raises(AssertionError):
        MoECUDA(k=5)(x, r, g, d)                        # more choices than experts
    with pytest.raises(RuntimeError, match="backward"):
        layer(x.requires_grad_(), r, g, d)
    x, r, g, d = operands()
    with pytest.raises(RuntimeError, match="backward"):
        layer(x, r, g.requires_grad_(), d)


def test_four_bit_experts_refusals():
    def four(w):
        codes, scales = _mx4.encode(w.float().numpy())
        return MX4Tensor.from_blocks(torch.from_numpy(_mx4.packed(codes)), torch.from_numpy(scales), w.shape[-1])
    layer = MoECUDA(k=2)
    x, r, g, d = operands()
    for args in ((x, r, four(g), d), (x, r, g, four(d)), (x, r, four(g), four(d.transpose(1, 2).contiguous()).transpose(1, 2)),
                 (x, r, four(g[:, :, :32]), four(d)), (x, r, four(g), four(d))):
        with pytest.raises(AssertionError):
            layer(*args)


def desc(**kw):
    v = dict(T=3, H=64, I=32, E=4, k=2, x_dtype=_lib.BF16, router_dtype=_lib.BF16, w_dtype=_lib.BF16, activation=0,
             renormalize=1, ld_x=64, ld_router=64, ld_gate_up=64, stride_gate_up=4096, ld_down=32, stride_down=2048)
    v.update(kw)
    return _lib.MoeDesc(*[v[name] for name, _ in _lib.MoeDesc._fields_])


def test_desc_layout_matches_header():
    assert ctypes.sizeof(_lib.MoeDesc) == 10 * 4 + 6 * 8
    assert _lib.MoeDesc.ld_x.offset == 40


def test_refusals_of_the_c_entry_point():
    lib = _lib.load()
    p = ctypes.c_void_p(0x1000)                          # never dereferenced

    def call(d, ptr=p, scales=None, ws=p, nbytes=1 << 30):
        return lib.cmk_moe(ptr, p, p, scales, p, scales, p, p, p, d, ws, nbytes, None)

    assert call(None) == _lib.ERR_INVALID_ARG
    for bad in (dict(T=-1), dict(H=0), dict(I=0), dict(E=0), dict(k=0), dict(k=5), dict(x_dtype=_lib.F32),
                dict(router_dtype=_lib.F16), dict(w_dtype=_lib.F16), dict(w_dtype=_lib.F32), dict(activation=2),
                dict(ld_x=63), dict(ld_router=63), dict(ld_gate_up=63), dict(ld_down=31), dict(stride_down=-1)):
        assert call(desc(**bad)) == _lib.ERR_INVALID_ARG, bad
        assert lib.cmk_moe_workspace_bytes(desc(**bad)) == 0
    for big in (dict(T=257), dict(E=1025), dict(E=64, k=33), dict(H=1 << 21, ld_x=1 << 21, ld_router=1 << 21, ld_gate_up=1 << 21)):
        assert call(desc(**big)) == _lib.ERR_UNSUPPORTED, big
    assert call(desc(), ptr=None) == _lib.ERR_INVALID_ARG
    assert call(desc(w_dtype=_lib.MX4)) == _lib.ERR_INVALID_ARG             # no scales
    assert call(desc(w_dtype=_lib.MX4), scales=ctypes.c_void_p(0x1002)) == _lib.ERR_INVALID_ARG
    assert call(desc(), ws=None) == _lib.ERR_WORKSPACE
    assert call(desc(), ws=ctypes.c_void_p(0x1010)) == _lib.ERR_WORKSPACE
    need = lib.cmk_moe_workspace_bytes(desc())
    assert need > 0 and call(desc(), nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert call(desc(T=0)) == 0                          # nothing to do


def test_extents_beyond_a_c_int_are_refused():
    """They would reach the library cut to 32 bits; meta tensors hold no elements."""
    def layer(h, i, e):
        def meta(*shape):
            return torch.empty(*shape, dtype=torch.bfloat16, device="meta")
        MoECUDA(k=1)(meta(3, h), meta(e, h), meta(e, 2 * i, h), meta(e, h, i))
    for large in (2 ** 31, 2 ** 32 + 64):
        for extents in ((large, 32, 4), (64, large, 4), (64, 32, large), (64, large // 2, 4)):
            with pytest.raises(ValueError, match="2\\^31"):
                layer(*extents)


def test_tangents_of_forward_mode_are_refused():
    import torch.autograd.forward_ad as forward_ad
    layer = MoECUDA(k=2)
    for n in range(4):
        args = list(operands())
        with forward_ad.dual_level():
            args[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer(*args)
