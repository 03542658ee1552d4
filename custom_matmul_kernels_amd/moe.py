"""A mixture-of-experts layer for a few tokens: router, choice, the chosen
experts' products and their weighted sum.  No counterpart in the reference; the
router is a top-k of a product and the experts are a routed batched product."""
import torch
from torch.autograd import forward_ad

from . import _common, _lib
from .mx4 import MX4Tensor

ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
CHUNK = 256        # tokens per library call


class MoECUDA:
    """``MoECUDA(k, activation, renormalize)(x, router, gate_up, down)`` returns
    (y, weights, experts).

    Per token the `k` experts of the largest x @ router.T (summed in 64 bits; the
    lowest index of equal ones, NaN above all) are weighted by the softmax of
    these over the chosen (`renormalize`) or over all experts, and
        y = sum_j weights_j * ((act(x @ gate.T) * (x @ up.T)) @ down_e.T)
    with gate and up the first and last i rows of gate_up[e].

    x: bfloat16 or float16 [t, h];  router: x's type or float32 [e, h]
    gate_up [e, 2i, h], down [e, h, i]: x's type with the last axis contiguous, or
    MX4Tensors of these shapes with blocks along the last axis
    returns y [t, h] in x's type, weights float32 [t, k], experts int64 [t, k]

    Made for a few tokens, where reading the chosen experts' weights is all there
    is; more than 256 run in portions of 256.  A y_j whose sum an infinite weight of
    `down` or an infinite inner product enters may be NaN instead of an infinity.
    There is no backward pass and no forward-mode derivative: operands that ask for
    one are refused."""

    def __init__(self, k=2, activation="silu", renormalize=True):
        if activation not in ACTIVATIONS:
            raise ValueError("Unrecognized activation")
        assert type(renormalize) == bool
        assert k >= 1
        self.k, self.activation, self.renormalize = k, activation, renormalize
        self._activation = ACTIVATIONS[activation]
        self._lib = _lib.load()

    @staticmethod
    def _experts(W, shape, dtype, name):
        """[e, r, c] weights, to be kept until the launch, and their (pointer, scales'
        pointer, row stride, expert stride)."""
        if isinstance(W, MX4Tensor):
            assert W.shape == shape
            assert W.k_axis == -1, "the blocks of %s must run along its last axis" % name
            return W, W._pointers() + (0, 0)
        if W.dtype != dtype:
            raise TypeError("%s must be an MX4Tensor or of x's type, got %s" % (name, W.dtype))
        assert W.shape == shape
        if W.requires_grad or forward_ad._current_level >= 0:
            _common.refuse_grad(W)
        if W.is_neg():
            W = _common.with_own_sign(W)
        e, r, c = shape
        s0, s1, s2 = W.stride()
        if (s2 != 1 and c > 1) or (s1 < c and r > 1):
            raise ValueError("the last axis of %s must be contiguous" % name)
        return W, (W.data_ptr(), None, s1 if r > 1 else c, s0 if e > 1 else 0)

    def __call__(self, x, router, gate_up, down):
        dtype, device = x.dtype, x.device
        if dtype != torch.bfloat16 and dtype != torch.float16:
            raise TypeError("x must be torch.bfloat16 or torch.float16, got %s" % dtype)
        if router.dtype != dtype and router.dtype != torch.float32:
            raise TypeError("router must be torch.float32 or of x's type, got %s" % router.dtype)
        if x.dim() != 2 or router.dim() != 2 or gate_up.dim() != 3 or down.dim() != 3:
            raise ValueError("x and router need to be 2d, gate_up and down 3d")
        t, h = x.shape
        e, two_i, _ = gate_up.shape
        i = two_i // 2
        assert router.shape == (e, h)
        assert two_i == 2 * i and i > 0 and h > 0
        assert 0 < self.k <= e
        if e | two_i | h > _common.MAX_EXTENT:
            _common.check_extents(e, two_i, h)
        if x.requires_grad or router.requires_grad or forward_ad._current_level >= 0:
            _common.refuse_grad(x, router)
        gate_up, (gp, gs, ldg, sg) = self._experts(gate_up, (e, two_i, h), dtype, "gate_up")
        down, (dp, ds, ldd, sd) = self._experts(down, (e, h, i), dtype, "down")
        assert (gs is None) == (ds is None), "gate_up and down must be of one kind"
        assert device.type == "cuda"
        assert router.device == device and gate_up.device == device and down.device == device
        if x.is_neg() or router.is_neg():
            x, router = _common.with_own_sign(x), _common.with_own_sign(router)
        sx, sr = x.stride(), router.stride()
        if h > 1 and sx[1] != 1 or t > 1 and sx[0] < h:
            x = x.contiguous()
            sx = (h, 1)
        if h > 1 and sr[1] != 1 or e > 1 and sr[0] < h:
            router = router.contiguous()
            sr = (h, 1)
        y = torch.empty((t, h), dtype=dtype, device=device)
        weights = torch.empty((t, self.k), dtype=torch.float32, device=device)
        experts = torch.empty((t, self.k), dtype=torch.int64, device=device)
        code = _common.FLOAT_TYPES[dtype]
        rest = (h, i, e, self.k, code, _common.FLOAT_TYPES[router.dtype], code if gs is None else _lib.MX4,
                self._activation, int(self.renormalize), max(sx[0], h), max(sr[0], h), ldg, sg, ldd, sd)
        for t0 in range(0, t, CHUNK):
            d = _lib.MoeDesc(min(CHUNK, t - t0), *rest)
            part = (x, y, weights, experts) if t0 == 0 else (x[t0:], y[t0:], weights[t0:], experts[t0:])
            _common.call_with_workspace(self._lib.cmk_moe_workspace_bytes, self._lib.cmk_moe, device, (d,),
                                        (part[0].data_ptr(), router.data_ptr(), gp, gs, dp, ds, part[1].data_ptr(),
                                         part[2].data_ptr(), part[3].data_ptr(), d))
        return y, weights, experts
