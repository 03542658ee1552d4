"""Mixture-of-experts layer on the GPU against the formulas in 64 bits.

The choice has one right answer.  Outputs: fp32 sums of H and I products are off
by at most n * 2^-23 * sum |.| (any order, rounding or truncating adders), the
activation by a few steps, the kept inner values by 2^-16 (two bf16; in front of
fp16 weights, which are split too, the smallest of the four partial products is
left out: 2^-16 more), y by half a step of its type.  The bound is carried through the
formula in 64 bits, element by element.  (It is the bound of inner values of 16 bits; they
have 24, which layers with an exact result check to the bit.)"""
import math

import pytest
import torch

import _mx4
from custom_matmul_kernels_amd import MoECUDA, quantize_mx4

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -23


def make(t, h, i, e, dtype, seed, router_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, generator=gen)
    x[:, ::29] *= 8
    return (x.to(dtype), (torch.randn(e, h, generator=gen) * h ** -0.5).to(router_dtype or dtype),
            (torch.randn(e, 2 * i, h, generator=gen) * h ** -0.5).to(dtype),
            (torch.randn(e, h, i, generator=gen) * i ** -0.5).to(dtype))


def act64(g, name):
    return g / (1 + torch.exp(-g)) if name == "silu" else g * 0.5 * (1 + torch.erf(g / math.sqrt(2)))


def reference(x, router, gate_up, down, k, activation, renormalize):
    """y, its error bound before the last rounding, weights, experts; all in float64."""
    x, router, gate_up, down = (v.double() for v in (x, router, gate_up, down))
    t, h = x.shape
    i = down.shape[2]
    score = torch.stack([(x[j] * router).sum(1) for j in range(t)])
    experts = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k]
    picked = score.gather(1, experts)
    weights = torch.softmax(picked, 1) if renormalize else torch.softmax(score, 1).gather(1, experts)
    spread = (picked - picked[:, :1]).abs()
    d_weights = weights * (spread + 16 + score.shape[1]) * U
    y, dy = torch.zeros(t, h, dtype=torch.float64), torch.zeros(t, h, dtype=torch.float64)
    for e in experts.unique().tolist():
        rows, j = (experts == e).nonzero(as_tuple=True)
        G, V, D = gate_up[e, :i], gate_up[e, i:], down[e]
        xr = x[rows]
        g, v = xr @ G.t(), xr @ V.t()
        # an fp16 x in front of 4-bit weights is two products an element
        dg, dv = 2 * h * U * (xr.abs() @ G.abs().t()), 2 * h * U * (xr.abs() @ V.abs().t())
        a = act64(g, activation)
        da = 1.13 * dg + 8 * U * (a.abs() + g.abs())
        m = a * v
        dm = da * v.abs() + a.abs() * dv + da * dv + m.abs() * 2.0 ** -16
        z = m @ D.t()
        dz = dm @ D.abs().t() + (3 * i * U + 2.0 ** -16) * ((m.abs() + dm) @ D.abs().t())
        w, dw = weights[rows, j][:, None], d_weights[rows, j][:, None]
        y[rows] += w * z
        dy[rows] += (w + dw) * dz + dw * z.abs() + k * U * w * z.abs()
    return y, dy, weights, d_weights, experts


def check(layer, x, router, gate_up, down, device, four_bit):
    print("moe", tuple(x.shape), tuple(gate_up.shape), layer.k, x.dtype, "mx4" if four_bit else "plain", flush=True)
    if four_bit:
        gd, dd = quantize_mx4(gate_up.to(device)), quantize_mx4(down.to(device))
        gate_up, down = _mx4.rounded(gate_up), _mx4.rounded(down)
    else:
        gd, dd = gate_up.to(device), down.to(device)
    got = layer(x.to(device), router.to(device), gd, dd)
    y, dy, weights, d_weights, experts = reference(x, router, gate_up, down, layer.k, layer.activation, layer.renormalize)
    assert got[0].dtype == x.dtype and got[1].dtype == F32 and got[2].dtype == torch.int64
    assert torch.equal(got[2].cpu(), experts)
    assert ((got[1].cpu().double() - weights).abs() <= d_weights + 1e-37).all()
    fi = torch.finfo(x.dtype)
    bound = dy + (y.abs() + dy) * fi.eps / 2 + fi.smallest_normal * fi.eps
    off = (got[0].cpu().double() - y).abs()
    assert (off <= bound).all(), "off by %g of the bound" % (off / bound).max()
    return got


SHAPES = [(1, 64, 32, 4, 2), (1, 1, 1, 1, 1), (1, 100, 33, 10, 3), (2, 256, 130, 6, 6), (7, 1000, 333, 10, 3),
          (16, 256, 128, 8, 2), (17, 130, 257, 70, 5), (70, 96, 48, 3, 3), (200, 72, 40, 2, 1), (40, 64, 64, 130, 8),
          (5, 2048, 64, 33, 32), (3, 40, 1030, 9, 4), (33, 128, 300, 300, 3),
          # many tokens an expert: up to 16, up to 32, more
          (100, 512, 512, 32, 2), (130, 700, 530, 32, 2), (200, 640, 520, 32, 8), (100, 1300, 513, 32, 2)]


@pytest.mark.parametrize("t,h,i,e,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("four_bit", [False, True])
def test_layer(device, t, h, i, e, k, dtype, four_bit):
    check(MoECUDA(k=k), *make(t, h, i, e, dtype, t + h + i), device, four_bit)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("router_dtype", [None, F32])
def test_options(device, activation, renormalize, router_dtype):
    for dtype, four_bit in ((BF16, False), (F16, True), (F16, False), (BF16, True)):
        check(MoECUDA(k=3, activation=activation, renormalize=renormalize),
              *make(9, 160, 70, 12, dtype, 3, router_dtype), device, four_bit)


def test_more_tokens_than_one_call_takes(device):
    check(MoECUDA(k=2), *make(300, 64, 32, 5, BF16, 1), device, False)
    y, weights, experts = MoECUDA(k=2)(*(v.to(device) for v in make(0, 64, 32, 5, BF16, 1)))
    assert y.shape == (0, 64) and weights.shape == (0, 2) and experts.shape == (0, 2)


def test_equal_logits_go_to_the_lowest_index(device):
    x, router, gate_up, down = make(6, 96, 40, 12, BF16, 5)
    router[7] = router[2]
    router[11] = router[2]
    router[4] = router[9]
    check(MoECUDA(k=7), x, router, gate_up, down, device, False)
    router[:] = 0
    got = check(MoECUDA(k=5), x, router, gate_up, down, device, True)
    assert (got[2].cpu() == torch.arange(5)).all() and (got[1] == 0.2).all()


def test_close_logits_are_ordered_exactly(device):
    """Logits that differ by less than an fp32 sum could tell."""
    x, router, gate_up, down = make(4, 512, 32, 16, BF16, 6)
    router[:] = router[:1]
    for e in range(16):
        router[e, e * 31] += 2.0 ** -10 * ((e * 7) % 16 - 8)
    check(MoECUDA(k=8), x, router, gate_up, down, device, False)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_nan_and_infinity_stay_where_they_belong(device, four_bit, dtype):
    x, router, gate_up, down = make(20, 200, 70, 9, dtype, 7)
    layer = MoECUDA(k=3)
    want = check(layer, x, router, gate_up, down, device, four_bit)
    def run(x, gate_up, down):
        if four_bit:
            gate_up, down = quantize_mx4(gate_up.to(device)), quantize_mx4(down.to(device))
        return layer(x.to(device), router.to(device), *(v if four_bit else v.to(device) for v in (gate_up, down)))
    # a token with a NaN: its own row only; its choice is the first experts
    x2 = x.clone()
    x2[4, 17] = float("nan")
    y, w, e = run(x2, gate_up, down)
    assert torch.isnan(y[4]).all() and torch.isnan(w[4]).all() and e[4].tolist() == [0, 1, 2]
    keep = torch.arange(20) != 4
    assert torch.equal(y[keep], want[0][keep]) and torch.equal(e[keep], want[2][keep])
    # an expert with a NaN: the rows that chose it only
    bad = int(want[2][0, 0])
    g2, d2 = gate_up.clone(), down.clone()
    g2[bad, 5, 3] = float("nan")
    d2[bad, 9, 2] = float("inf")
    y, w, e = run(x, g2, d2)
    hit = (want[2] == bad).any(1)
    assert hit.any() and not hit.all()
    assert torch.equal(y[~hit], want[0][~hit]) and torch.equal(e, want[2])
    assert torch.isnan(y[hit]).all()


def test_inner_values_beyond_fp16(device):
    """act(g) * u of 1e6 and more: the layer's output still fits."""
    x, router, gate_up, down = make(5, 64, 40, 4, F16, 8)
    gate_up = (gate_up.float() * 500).half()
    down = (down.float() * 2.0 ** -12).half()
    check(MoECUDA(k=2), x, router, gate_up, down, device, False)
    check(MoECUDA(k=2), x, router, gate_up, down, device, True)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strided_operands(device, dtype):
    x, router, gate_up, down = make(11, 130, 45, 6, dtype, 9)
    layer = MoECUDA(k=2)
    want = check(layer, x, router, gate_up, down, device, False)
    def spread(v):     # rows and matrices apart from each other, at odd addresses
        shape = list(v.shape)
        shape[-1] += 5
        shape[0] += 1
        big = torch.full(shape, float("nan"), dtype=v.dtype, device=device)
        view = big[1:, ..., 3:3 + v.shape[-1]]
        view.copy_(v)
        return view
    got = layer(spread(x), spread(router), spread(gate_up), spread(down))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    got = layer(x.t().contiguous().t().to(device), router.t().contiguous().t().to(device), gate_up.to(device), down.to(device))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # all experts the same matrix, not copied
    one = check(layer, x, router, gate_up[:1].expand(6, 90, 130), down[:1].expand(6, 130, 45), device, False)
    got = layer(x.to(device), router.to(device), gate_up[:1].to(device).expand(6, 90, 130), down[:1].to(device).expand(6, 130, 45))
    assert torch.equal(got[0], one[0])


@pytest.mark.parametrize("t", [1, 30])
@pytest.mark.parametrize("four_bit", [False, True])
def test_streams_and_graphs(device, t, four_bit):
    x, router, gate_up, down = (v.to(device) for v in make(t, 192, 64, 16, BF16, 10))
    if four_bit:
        gate_up, down = quantize_mx4(gate_up), quantize_mx4(down)
    layer = MoECUDA(k=4)
    want = layer(x, router, gate_up, down)
    torch.cuda.synchronize()
    # two streams at once
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(layer(x, router, gate_up, down))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    # two graphs, replayed in turn with eager calls between
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, router, gate_up, down)
        graphs.append((graph, out))
    gen = torch.Generator().manual_seed(0)
    for step in range(4):
        x.copy_(torch.randn(t, 192, generator=gen))
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        for a, b in zip(got, layer(x, router, gate_up, down)):
            assert torch.equal(a, b), "replay %d differs" % step


def test_a_run_of_the_operators_together(device):
    """A decoding step as they would be used: a projection in 4 bits, the layer with
    4-bit experts on its result, and a 4-bit projection back."""
    from custom_matmul_kernels_amd import MX4BMMCUDA
    gen = torch.Generator().manual_seed(11)
    x = torch.randn(6, 96, generator=gen).to(BF16)
    w_in, w_out = torch.randn(96, 160, generator=gen) / 10, torch.randn(160, 50, generator=gen) / 13
    _, router, gate_up, down = make(6, 160, 64, 8, BF16, 12)
    inner = MX4BMMCUDA(out_dtype=BF16)(x.to(device), quantize_mx4(w_in.to(device), dim=-2))
    want = _mx4.rounded(x) @ _mx4.rounded(w_in.t()).t()
    assert torch.equal(inner.cpu(), want.to(BF16)) or (inner.cpu().double() - want).abs().max() <= want.abs().max() * 2.0 ** -8
    y, _, _ = check(MoECUDA(k=2), inner.cpu(), router, gate_up, down, device, True)
    out = MX4BMMCUDA()(y, quantize_mx4(w_out.to(device), dim=-2))
    a, b = _mx4.rounded(y), _mx4.rounded(w_out.t()).t()
    assert ((out.cpu().double() - a @ b).abs() <= 160 * U * (a.abs() @ b.abs())).all()


def test_offsets_beyond_32_bits(device):
    """4.7 GB and 2.3 GB of weights; the choice falls on the last experts."""
    e, h, i = 70, 4096, 4096
    gen = torch.Generator(device=device).manual_seed(2)
    gate_up = torch.empty(e, 2 * i, h, dtype=BF16, device=device).normal_(generator=gen).mul_(h ** -0.5)
    down = torch.empty(e, h, i, dtype=BF16, device=device).normal_(generator=gen).mul_(i ** -0.5)
    cpu = torch.Generator().manual_seed(3)
    x = torch.randn(2, h, generator=cpu).to(BF16)
    router = torch.randn(e, h, generator=cpu) * 1e-3
    router[e - 1] = x[0].float()
    router[e - 2] = x[1].float()
    layer = MoECUDA(k=1)
    for t in (1, 2):
        y, weights, experts = layer(x[:t].to(device), router.to(device), gate_up, down)
        assert experts.flatten().tolist() == [e - 1, e - 2][:t]
        keep = [e - 1, e - 2]
        want, dy, _, _, _ = reference(x[:t], router[keep], gate_up[keep].cpu(), down[keep].cpu(), 1, "silu", True)
        assert ((y.cpu().double() - want).abs() <= dy + (want.abs() + dy) * 2.0 ** -8).all()


def test_results_do_not_change_from_run_to_run(device):
    args = [v.to(device) for v in make(64, 512, 256, 16, BF16, 13)]
    layer = MoECUDA(k=8)
    want = layer(*args)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(layer(*args), want))


def test_more_experts_than_are_ranked(device):
    """Beyond 256 experts the choice is made in rounds."""
    check(MoECUDA(k=9), *make(5, 130, 40, 300, BF16, 14), device, False)
    check(MoECUDA(k=32, renormalize=False), *make(1, 64, 32, 1024, F16, 15), device, True)
    x, router, gate_up, down = make(3, 64, 32, 700, BF16, 16)
    router[650] = router[3]
    router[20] = router[3]
    x[1, 5] = float("nan")
    y, w, e = MoECUDA(k=6)(*(v.to(device) for v in (x, router, gate_up, down)))
    assert e[1].tolist() == [0, 1, 2, 3, 4, 5] and torch.isnan(y[1]).all()
    check(MoECUDA(k=6), x[::2], router, gate_up, down, device, False)


@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinite_down_weight_reaches_its_own_feature_only(device, t, dtype):
    x, router, gate_up, down = make(t, 200, 70, 9, dtype, 7)
    x, router, gate_up, down = (v.to(device) for v in (x, router, gate_up, down))
    layer = MoECUDA(k=3)
    want = layer(x, router, gate_up, down)
    bad = int(want[2][0, 0])
    down[bad, 9, 2] = float("inf")
    y, w, e = layer(x, router, gate_up, down)
    hit = (want[2] == bad).any(1)
    assert torch.equal(e, want[2]) and torch.equal(w, want[1])
    assert not torch.isfinite(y[hit, 9]).any()
    y[hit, 9] = want[0][hit, 9]
    assert torch.equal(y, want[0])


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_equal_tokens_get_equal_results(device, four_bit, dtype):
    """237 slots of one expert: the kernels take them in passes of up to 32, in an order
    that may change from run to run, and the last pass is a smaller one."""
    x, router, gate_up, down = make(1, 700, 700, 64, dtype, 15)
    gate_up, down = gate_up.to(device), down.to(device)
    if four_bit:
        gate_up, down = quantize_mx4(gate_up), quantize_mx4(down)
    y, w, e = MoECUDA(k=1)(x.to(device).expand(237, 700), router.to(device), gate_up, down)
    assert (e == e[0]).all() and torch.equal(y, y[:1].expand_as(y))


@pytest.mark.parametrize("t,h,i,e,k,dtype", [(130, 1000, 260, 64, 4, F16), (100, 2040, 300, 64, 4, BF16), (180, 2044, 260, 64, 8, F16)])
def test_many_tokens_of_many_experts_in_four_bits(device, t, h, i, e, k, dtype):
    """Two and four groups of rows a wave, with up to 16, up to 32 and more slots."""
    check(MoECUDA(k=k), *make(t, h, i, e, dtype, t + h + i), device, True)


def exact_layer(t, e, h, i):
    """Operands (bf16) whose layer has an exact result, and that result in float64.

    g = 32 for every inner feature: 1 + exp(-32) is 1 in fp32, so silu(g) = 32 there.
    Up values are 1 + a sum of distinct powers of two down to 2^-23, products of powers of
    two; every row of `down` is the difference of two inner values.  All of that and the
    choice (equal logits: the first two experts, half each) is exact in fp32 whatever the
    order of the sums, as long as inner values have 24 bits."""
    gen = torch.Generator().manual_seed(t)
    blocks = torch.arange(0, h, 32)[:14]               # one element a block of 32: exact in 4 bits
    low = blocks[1:]
    power = torch.arange(1, 14) + 10                   # 2^-11 to 2^-23
    x = torch.zeros(t, h)
    x[:, 0] = 1
    x[:, low] = torch.randint(0, 2, (t, 13), generator=gen) * 2.0 ** -10
    x[0, low] = 2.0 ** -10
    gate_up, down = torch.zeros(e, 2 * i, h), torch.zeros(e, h, i)
    gate_up[:, :i, 0] = 32
    gate_up[:, i:, 0] = 1
    gate_up[:, i:, low] = torch.randint(0, 2, (e, i, 13), generator=gen) * torch.exp2(10.0 - power)
    minus = (torch.arange(h) * 7 + 3) % i
    plus = torch.where((torch.arange(h) * 5) % i == minus, (minus + 1) % i, (torch.arange(h) * 5) % i)
    down[:, torch.arange(h), plus], down[:, torch.arange(h), minus] = 1, -1
    v = x.double() @ gate_up[:2, i:].double().transpose(1, 2)                       # [2, t, i]
    y = ((32 * v) @ down[:2].double().transpose(1, 2) * 0.5).sum(0)
    return x, torch.zeros(e, h), gate_up, down, y


# one token; planes in one and in two fragments of their own; one and two blocks of slots;
# passes; the ring of activations
@pytest.mark.parametrize("t,e,size", [(1, 4, 512), (2, 4, 512), (5, 8, 512), (6, 4, 512), (10, 8, 512), (11, 8, 512), (16, 40, 512),
                                      (25, 4, 512), (25, 16, 512), (40, 40, 512), (100, 32, 512), (200, 32, 1024), (240, 33, 1000)])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_inner_values_keep_their_24_bits(device, t, e, size, four_bit, dtype):
    x, router, gate_up, down, want = exact_layer(t, e, size, size)
    print("exact layer", t, e, size, four_bit, dtype, flush=True)
    args = [v.to(dtype).to(device) for v in (x, router, gate_up, down)]
    for v, w in zip((x, gate_up, down), (args[0], args[2], args[3])):
        assert torch.equal(w.cpu().float(), v)
    if four_bit:
        args[2:] = [quantize_mx4(v) for v in args[2:]]
        for v, w in zip((gate_up, down), args[2:]):
            assert torch.equal(w.dequantize().cpu(), v)
    y, weights, experts = MoECUDA(k=2)(*args)
    assert (weights == 0.5).all() and (experts.cpu() == torch.tensor([0, 1])).all()
    assert want[0].abs().min() < 2.0 ** -7 < want[0].abs().max()      # far below the inner values' 32
    assert torch.equal(y.cpu(), want.to(dtype))


@pytest.mark.parametrize("t,e", [(1, 4), (4, 8), (14, 8), (20, 4), (20, 16), (40, 40), (100, 32)])
@pytest.mark.parametrize("four_bit", [False, True])
def test_inner_values_at_the_end_of_the_range(device, t, e, four_bit):
    """2^128 (1 - 2^-12) is finite, and the nearest bf16 is not: g = 2^64, up 2^64 - 2^52."""
    h = i = 512
    x, gate_up, down = torch.zeros(t, h), torch.zeros(e, 2 * i, h), torch.zeros(e, h, i)
    x[:, 0], x[:, 64] = 2.0 ** 32, 2.0 ** 20
    gate_up[:, :, 0] = 2.0 ** 32
    gate_up[:, i:, 64] = -2.0 ** 32
    down[:, torch.arange(h), torch.arange(h)] = 2.0 ** -100
    args = [v.to(BF16).to(device) for v in (x, torch.zeros(e, h), gate_up, down)]
    if four_bit:
        args[2:] = [quantize_mx4(v) for v in args[2:]]
        assert torch.equal(args[3].dequantize().cpu(), down)
    y, _, _ = MoECUDA(k=2)(*args)
    assert (y == 2.0 ** 28).all()        # 2^28 (1 - 2^-12), rounded


def check_grouped(sizes, h, i, e, dtype, four_bit, device):
    """A layer of e experts whose expert j is the choice of sizes[j] tokens, in a shuffled
    order; the other experts (zeros) are nobody's."""
    print("grouped", sizes, h, i, e, dtype, four_bit, flush=True)
    n, t = len(sizes), sum(sizes)
    x, router, gate_up, down = make(t, h, i, n, dtype, h + i)
    choice = torch.cat([torch.full((s,), j) for j, s in enumerate(sizes)])
    choice = choice[torch.randperm(t, generator=torch.Generator().manual_seed(h))]
    x[:, :n] = 0
    x[torch.arange(t), choice] = 6
    router[:, :n] = 8 * torch.eye(n)
    def padded(v):
        return torch.cat([v.to(device), torch.zeros((e - n,) + v.shape[1:], dtype=dtype, device=device)])
    args = [x.to(device), padded(router), padded(gate_up), padded(down)]
    if four_bit:
        args[2:] = [quantize_mx4(v) for v in args[2:]]
        gate_up, down = _mx4.rounded(gate_up), _mx4.rounded(down)
    y, weights, experts = MoECUDA(k=1)(*args)
    assert torch.equal(experts.cpu()[:, 0], choice) and (weights == 1).all()
    want, dy, _, _, chosen = reference(x, router, gate_up, down, 1, "silu", True)
    assert torch.equal(chosen[:, 0], choice)
    fi = torch.finfo(dtype)
    off = (y.cpu().double() - want).abs()
    assert (off <= dy + (want.abs() + dy) * fi.eps / 2 + fi.smallest_normal * fi.eps).all()


# Slots of an expert decide how its rows are multiplied: planes packed in one fragment of
# columns (up to 5) or two (up to 10), blocks of 16 and of 32, passes of 32; the extents
# decide in how many pieces k goes through LDS, and by how many waves.
@pytest.mark.parametrize("sizes,h,i,e", [
    ((5, 9, 14, 27, 40), 1700, 1700, 16),    # few experts: waves share k in both products
    ((5, 9, 14, 27, 40), 3700, 300, 16),
    ((4, 10, 16, 32, 33), 300, 3700, 16),
    ((6, 2), 4200, 1400, 9),                 # fewer slots than experts
    ((5, 9, 14, 27, 40), 520, 1300, 33),     # more than 32 experts: rows of their own
    ((4, 8, 16, 32, 49), 2300, 260, 33),
    ((5, 9, 14, 27, 40), 1100, 700, 5),      # the ring of activations in 4 bits
    ((3, 17, 33, 64), 130, 1500, 4),
])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("four_bit", [False, True])
def test_experts_of_every_size(device, sizes, h, i, e, dtype, four_bit):
    check_grouped(sizes, h, i, e, dtype, four_bit, device)


@pytest.mark.parametrize("t,h,i,e,k", [(200, 1024, 1100, 32, 2), (240, 821, 830, 40, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_tokens_of_many_large_experts(device, t, h, i, e, k, dtype):
    """The ring of activations in 16 bits, one and two groups of rows a wave; four experts
    are most tokens' choice, the others have a few slots."""
    x, router, gate_up, down = make(t, h, i, e, dtype, t)
    check(MoECUDA(k=k), x, router, gate_up, down, device, False)
    x[:, 0] = 2
    router[:4, 0] = 2
    got = check(MoECUDA(k=k), x, router, gate_up, down, device, False)
    count = got[2].flatten().bincount(minlength=e)
    assert count.max() > 64 and 0 < count[4:].max() <= 16


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_negated_views_are_read_with_their_sign(device, dtype):
    args = [v.to(device) for v in make(5, 96, 40, 6, dtype, 17)]
    layer = MoECUDA(k=2)
    want = layer(*args)
    for n in range(4):
        some = list(args)
        some[n] = torch._neg_view(-args[n])
        assert some[n].is_neg() and torch.equal(some[n], args[n])
        assert all(torch.equal(a, b) for a, b in zip(layer(*some), want))
