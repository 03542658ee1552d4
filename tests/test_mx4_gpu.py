"""4-bit microscaled matrices on the GPU against the definition in 64 bits.

Quantisation has one right answer: codes and scales are compared bit by bit.
Products: the values are exact, so an output is off by the fp32 accumulation, at
most k * 2^-23 * sum |a b| for any order of the sums and rounding or truncating
adders, plus half a step of the output type."""
import numpy as np
import pytest
import torch

import _mx4
from custom_matmul_kernels_amd import MX4BMMCUDA, MX4Tensor, quantize_mx4

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def normal(shape, seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    x[..., ::37] *= 20
    return x.to(dtype)


def check_blocks(x, q):
    """x: host tensor [l, rows, k]; q: MX4Tensor on the device."""
    print("blocks", tuple(x.shape), x.dtype, flush=True)
    codes, scales = _mx4.encode(x.double().numpy())
    got_c, got_s = q.blocks()
    if q.two_dimensional:
        got_c, got_s = got_c[None], got_s[None]
    assert np.array_equal(got_s.cpu().numpy(), scales)
    assert np.array_equal(got_c.cpu().numpy(), _mx4.packed(codes))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("l,rows,k", [(1, 1, 1), (1, 1, 32), (2, 3, 31), (1, 17, 33), (3, 16, 128), (2, 65, 129),
                                      (1, 100, 1000), (2, 130, 520), (1, 7, 4097)])
def test_quantize_rows(device, dtype, l, rows, k):
    x = normal((l, rows, k), 1000 * rows + k, dtype)
    q = quantize_mx4(x.to(device))
    assert q.shape == (l, rows, k)
    check_blocks(x, q)
    # the padding up to a whole slab holds zero codes and zero scales
    tail = q.codes[:, -1].cpu()
    used = (k - 1) % 128 + 1
    assert (tail[:, :, (used + 1) // 2:] == 0).all()
    assert (q.scales[:, -1].cpu()[:, :, -(-used // 32):] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("l,rows,k", [(1, 1, 1), (2, 3, 31), (1, 65, 33), (3, 64, 128), (2, 130, 257), (1, 1000, 100)])
def test_quantize_columns(device, dtype, l, rows, k):
    """Blocks down the columns of a [k, rows] matrix."""
    x = normal((l, k, rows), 77 * rows + k, dtype)
    q = quantize_mx4(x.to(device), dim=1)
    assert q.shape == (l, k, rows) and q.k_axis == -2
    check_blocks(x.transpose(1, 2), q)


def test_quantize_strided_views(device):
    base = normal((4, 70, 300), 5).to(device)
    for view in (base[:, 3:50, 7:290], base[::2, ::3], base[:, :, ::2], base[:1].expand(3, 70, 300),
                 base.transpose(0, 1), base[:, :, 1:2], base[:, 5:6, :]):
        for dim in (-1, -2):
            q = quantize_mx4(view, dim=dim)
            x = view.cpu() if dim == -1 else view.cpu().transpose(1, 2)
            check_blocks(x, q)
    q = quantize_mx4(base[1], dim=0)
    assert q.shape == (70, 300)
    check_blocks(base[1].cpu().t()[None], q)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_special_values(device, dtype):
    """Ties, saturation, zero blocks, the ends of the exponent range, NaN and infinities."""
    fi = torch.finfo(dtype)
    rows = []
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.5, 7.0, 7.9, 0.2, 6.0, -0.25, -0.75, -5.0, -7.9])
    for scale in (1.0, 2.0 ** -8, 2.0 ** 5):
        rows.append(torch.cat([ties, -ties]) * scale)
    rows.append(torch.zeros(32))
    rows.append(torch.full((32,), -0.0))
    rows.append(torch.full((32,), fi.max))
    rows.append(torch.full((32,), fi.tiny))
    rows.append(torch.arange(32) * fi.smallest_normal / 7)
    rows.append(torch.arange(32) * float(np.finfo(np.float32).smallest_subnormal) * 3.0)
    rows.append(torch.arange(32) * 2.0 ** -130)
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.ones(32)
        r[11] = bad
        rows.append(r)
    x = torch.stack(rows).to(dtype)
    q = quantize_mx4(x.to(device))
    check_blocks(x[None], q)
    # the same columns-wise
    q = quantize_mx4(x.t().contiguous().to(device), dim=0)
    check_blocks(x[None], q)
    v = q.dequantize().cpu().t()
    want = _mx4.rounded(x)
    assert torch.equal(torch.isnan(v), torch.isnan(want))
    assert torch.isnan(v).all(1).sum() == 3
    fine = ~torch.isnan(want)
    assert torch.equal(v.double()[fine], want[fine])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k_axis", [-1, -2])
def test_dequantize(device, dtype, k_axis):
    for l, rows, k in ((1, 1, 1), (2, 33, 70), (3, 65, 129), (1, 200, 512), (2, 5, 1001)):
        x = normal((l, rows, k), k)
        want = _mx4.rounded(x)
        q = quantize_mx4(x.to(device))
        if k_axis == -2:
            q, want = q.transpose(), want.transpose(1, 2)
        got = q.dequantize(dtype)
        assert got.shape == q.shape and got.is_contiguous()
        assert torch.equal(got.cpu(), want.to(dtype))


def check_product(got, a, b, dtype):
    """a [l, m, k], b [l, k, n] in float64, the 4-bit values."""
    assert got.dtype == dtype
    want, size = a @ b, a.abs() @ b.abs()
    k = a.shape[2]
    bound = size * (k * 2.0 ** -23) + want.abs() * (torch.finfo(dtype).eps / 2) * (1 + k * 2.0 ** -23) \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.cpu().double() - want).abs()
    assert got.shape == want.shape
    assert (off <= bound).all(), "off by %g of the bound" % (off / bound).max()


SHAPES = [(1, 1, 1, 1), (1, 1, 17, 32), (2, 5, 3, 100), (1, 16, 64, 128), (3, 33, 65, 129), (1, 128, 128, 256),
          (2, 130, 200, 300), (1, 257, 129, 1000), (1, 1, 500, 4096), (1, 64, 1000, 640), (1, 40, 31, 5000),
          (1, 300, 513, 130), (5, 20, 20, 20), (1, 513, 700, 2050),
          # each tile, with edges, odd widths and every remainder of the ring of slabs
          (1, 100, 70, 1100), (1, 100, 70, 1030), (1, 100, 71, 800), (1, 100, 70, 700), (1, 100, 70, 600), (1, 100, 70, 513),
          (1, 65, 64, 300), (1, 100, 70, 1), (64, 200, 150, 300), (64, 200, 151, 640), (64, 260, 300, 130), (64, 257, 259, 900),
          # a contraction cut into ranges
          (1, 130, 96, 5000), (2, 70, 101, 9000), (1, 200, 333, 2300)]


@pytest.mark.parametrize("l,m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_product(device, dtype, l, m, n, k):
    print("product", (l, m, n, k), dtype, flush=True)
    x, w = normal((l, m, k), m + k, dtype), normal((l, k, n), n + k)
    A, B = quantize_mx4(x.to(device)), quantize_mx4(w.to(device), dim=-2)
    a, b = _mx4.rounded(x), _mx4.rounded(w.transpose(1, 2)).transpose(1, 2)
    got = MX4BMMCUDA(out_dtype=dtype)(A, B)
    check_product(got, a, b, dtype)
    # quantised in the call: the same bits
    for left, right in ((x.to(device), B), (A, w.to(device)), (x.to(device), w.to(device))):
        assert torch.equal(MX4BMMCUDA(out_dtype=dtype)(left, right), got)


def test_product_two_dimensions_and_views(device):
    x, w = normal((70, 300), 1).to(device), normal((300, 90), 2).to(device)
    product = MX4BMMCUDA()
    got = product(x, quantize_mx4(w, dim=0))
    assert got.shape == (70, 90)
    check_product(got[None], _mx4.rounded(x)[None], _mx4.rounded(w.t()).t()[None], torch.float32)
    # any strides of a float operand
    base = normal((3, 40, 520), 3).to(device)
    for left in (base[:, ::2, 5:305], base[:, :20, ::2][:, :, :150], base[:1, :9, :300].expand(3, 9, 300),
                 base[:, :, :33].transpose(1, 2)[:, :, :40]):
        k = left.shape[2]
        right = normal((3, 50, k), k).to(device)
        got = product(left, right.transpose(1, 2))
        check_product(got, _mx4.rounded(left), _mx4.rounded(right).transpose(1, 2), torch.float32)


def test_product_with_an_empty_axis(device):
    product = MX4BMMCUDA()
    assert product(torch.zeros(2, 0, 40, device=device), torch.zeros(2, 40, 3, device=device)).shape == (2, 0, 3)
    assert product(torch.zeros(0, 4, 40, device=device), torch.zeros(0, 40, 3, device=device)).shape == (0, 4, 3)
    assert product(torch.zeros(2, 4, 40, device=device), torch.zeros(2, 40, 0, device=device)).shape == (2, 4, 0)
    got = product(torch.zeros(2, 4, 0, device=device), torch.zeros(2, 0, 3, device=device))
    assert got.shape == (2, 4, 3) and (got == 0).all()
    assert quantize_mx4(torch.zeros(2, 0, 40, device=device)).dequantize().shape == (2, 0, 40)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_nan_stays_in_its_row(device, m):
    x, w = normal((1, m, 200), 1), normal((1, 200, 70), 2)
    x[0, m // 2, 150] = float("nan")
    w[0, 20, 33] = float("inf")
    got = MX4BMMCUDA()(x.to(device), quantize_mx4(w.to(device), dim=-2)).cpu()
    bad = torch.zeros(1, m, 70, dtype=torch.bool)
    bad[0, m // 2] = True
    bad[0, :, 33] = True
    assert torch.equal(torch.isnan(got), bad)


def test_large_and_small_scales(device):
    """Block scales far apart: the sums keep fp32's range."""
    x, w = normal((1, 20, 256), 1), normal((1, 256, 40), 2)
    x[..., :32] *= 2.0 ** 40
    x[..., 32:64] *= 2.0 ** -60
    w[:, 32:64] *= 2.0 ** 50
    got = MX4BMMCUDA()(x.to(device), w.to(device))
    check_product(got, _mx4.rounded(x), _mx4.rounded(w.transpose(1, 2)).transpose(1, 2), torch.float32)


def test_on_another_stream(device):
    x, w = normal((1, 5, 1000), 1).to(device), normal((1, 1000, 300), 2).to(device)
    want = MX4BMMCUDA()(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [MX4BMMCUDA()(x, w) for _ in range(3)]
    side.synchronize()
    for g in got:
        assert torch.equal(g, want)


@pytest.mark.parametrize("m", [1, 16, 200])
def test_replays_in_a_graph(device, m):
    x, w = normal((1, m, 600), 1).to(device), normal((1, 600, 300), 2).to(device)
    B = quantize_mx4(w, dim=-2)
    product = MX4BMMCUDA(out_dtype=torch.bfloat16)
    product(x, B)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = product(x, B)
    for step in range(3):
        x.copy_(normal((1, m, 600), 10 + step))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, product(x, B)), "replay %d differs" % step


def test_offsets_beyond_32_bits(device):
    """18 GB of elements, 4.8 GB of codes: rows far apart against the definition."""
    rows, k = 140000, 65536
    gen = torch.Generator(device=device).manual_seed(1)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=device).normal_(generator=gen)
    q = quantize_mx4(x)
    for r in (0, 70001, rows - 1):
        codes, scales = _mx4.encode(x[r].cpu().double().numpy())
        got = torch.stack((q.codes[0, :, r] & 15, q.codes[0, :, r] >> 4), -1).flatten().cpu().numpy()
        assert np.array_equal(got, codes)
        assert np.array_equal(q.scales[0, :, r].flatten().cpu().numpy(), scales)
    some = torch.tensor([0, 1, 32767, 32768, 70001, 139998, rows - 1])
    b = _mx4.rounded(x[some.to(device)])
    for m in (3, 40):                                    # by rows and by tiles
        a = normal((m, k), m)
        got = MX4BMMCUDA()(a.to(device), q.transpose())[:, some.to(device)]
        check_product(got[None], _mx4.rounded(a)[None], b.t()[None], torch.float32)
    del q
    back = quantize_mx4(x.t(), dim=0).dequantize(torch.bfloat16)      # [k, rows], blocks down the columns
    assert torch.equal(back[:, some.to(device)].cpu().double(), b.t())


def test_small_results_keep_their_values(device):
    """Products around and below the smallest normal fp32 number."""
    x, w = normal((1, 20, 256), 1) * 2.0 ** -60, normal((1, 256, 40), 2) * 2.0 ** -64
    a, b = _mx4.rounded(x), _mx4.rounded(w.transpose(1, 2)).transpose(1, 2)
    for m in (20, 3):
        check_product(MX4BMMCUDA()(x[:, :m].to(device), w.to(device)), a[:, :m], b, torch.float32)
    x = x * 2.0 ** -6                                    # results of 2^-130 to 2^-126
    got = MX4BMMCUDA()(x.to(device), w.to(device)).cpu().double()
    want = _mx4.rounded(x) @ b
    assert ((got - want).abs() <= torch.finfo(torch.float32).smallest_normal).all()      # flushed or not


def test_the_same_tensor_on_both_sides(device):
    x = normal((2, 150, 300), 4).to(device)
    a = _mx4.rounded(x)
    check_product(MX4BMMCUDA()(x, x.transpose(1, 2)), a, a.transpose(1, 2), torch.float32)
    q = quantize_mx4(x)
    assert torch.equal(MX4BMMCUDA()(q, q.transpose()), MX4BMMCUDA()(x, x.transpose(1, 2)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_results_past_the_caches(device, dtype):
    """Results of 32 MB and more, and just less, take different stores."""
    for l, m, n in ((1, 4096, 4096), (3, 1000, 4224), (1, 4096, 4095)):
        x, w = normal((l, m, 130), 1, dtype).to(device), normal((l, 130, n), 2, dtype).to(device)
        got = MX4BMMCUDA(out_dtype=dtype)(x, w)
        rows = torch.tensor([0, 1, m // 2, m - 1], device=device)
        check_product(got[:, rows], _mx4.rounded(x[:, rows]), _mx4.rounded(w.transpose(1, 2)).transpose(1, 2), dtype)
    for dim in (-1, -2):
        x = normal((2, 2049, 4160), 3, dtype)
        got = quantize_mx4(x.to(device), dim=dim).dequantize(dtype).cpu()
        want = _mx4.rounded(x if dim == -1 else x.transpose(1, 2))
        assert torch.equal(got, (want if dim == -1 else want.transpose(1, 2)).to(dtype))


def test_as_many_matrices_as_a_launch_holds(device):
    """One row each; a few more would not fit a launch."""
    l = (1 << 24) - 1
    x = torch.ones(l, 1, 4, dtype=torch.bfloat16, device=device)
    x[-1] = 2.0
    x[l // 2] = 3.0
    a = quantize_mx4(x)
    b = quantize_mx4(x.transpose(1, 2), dim=-2)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    c = MX4BMMCUDA(torch.bfloat16)(a, b)
    want = torch.full((l, 1, 1), 4.0, dtype=torch.bfloat16, device=device)
    want[-1], want[l // 2] = 16.0, 36.0
    assert torch.equal(c, want)
    with pytest.raises(RuntimeError):
        MX4BMMCUDA(torch.bfloat16)(x[:1].expand(l + 1, 1, 4), x[:1].expand(l + 1, 1, 4).transpose(1, 2))


def test_negated_views_are_read_with_their_sign(device):
    """The imaginary part of a conjugate is a view whose memory has the other sign."""
    gen = torch.Generator().manual_seed(6)
    z = torch.complex(torch.randn(2, 20, 300, generator=gen), torch.randn(2, 20, 300, generator=gen)).to(device)
    for x in (z.conj().imag, torch._neg_view(z.real.contiguous().to(torch.bfloat16))):
        y = x.resolve_neg()
        assert x.is_neg() and not y.is_neg() and torch.equal(x, y)
        for dim in (-1, -2):
            a, b = quantize_mx4(x, dim=dim), quantize_mx4(y, dim=dim)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        product, kept = MX4BMMCUDA(), quantize_mx4(y)
        want = product(kept, kept.transpose())
        for left, right in ((x, x.transpose(1, 2)), (x, kept.transpose()), (kept, x.transpose(1, 2))):
            assert torch.equal(product(left, right), want)
        # few rows, quantised by the product
        assert torch.equal(product(x[:, :3], kept.transpose()), want[:, :3])
        one = quantize_mx4(y[:, :1])
        assert not torch.equal(product(one, kept.transpose()), product(quantize_mx4(-y[:, :1]), kept.transpose()))
