"""The operators of large language models that stand beside the batched products
- 4-bit microscaled floating point (quantisation, its inverse, the batched
product) and the mixture-of-experts layer for a few tokens - as measured cases:
in elementary torch operations, and as calls of this package.

``own`` says which of the two ``run`` computes."""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MX4_BYTES = 17 / 32            # 32 codes of 4 bits and one scale byte

# The midpoints of the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6; a value on one goes
# to the neighbour whose code is even.
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# Cost of the largest listed cases; drawn ones stay below.
MAX_ELEMENTS = 1 << 26
MAX_PRODUCT = 1 << 39
MAX_OUTPUT = 1 << 27
MAX_EXPERT_WEIGHTS = 128 * 3 * 2048 * 1024


def listed():
    return [
        # a few short vectors (keys of one step): nothing but launch latency
        dict(name="round_trip_small", op="round_trip", l=1, r=5, c=100, axis=-1, dtype="f32"),
        # the activations of a long prompt, blocks along the features
        dict(name="round_trip_activations", op="round_trip", l=1, r=8192, c=8192, axis=-1, dtype="bf16"),
        # a few weight matrices stored [k, n], blocks down the columns, odd width
        dict(name="round_trip_weights", op="round_trip", l=3, r=4096, c=4095, axis=-2, dtype="f32"),
        # one token through a square projection
        dict(name="product_token", op="product", l=1, m=1, n=4096, k=4096, a="bf16", b="mx4", out="bf16"),
        # a decoding batch through a wide projection
        dict(name="product_tokens", op="product", l=1, m=16, n=16384, k=8192, a="f16", b="mx4", out="f16"),
        # a ragged batch of products, both operands quantised in the call
        dict(name="product_ragged", op="product", l=3, m=333, n=777, k=1000, a="f32", b="f32", out="f32"),
        # the batched product of the package's own benchmark
        dict(name="product_batch", op="product", l=128, m=1024, n=1024, k=128, a="f32", b="f32", out="f32"),
        # a long prompt through a wide projection, weights kept in 4 bits
        dict(name="product_large", op="product", l=1, m=8192, n=8192, k=8192, a="bf16", b="mx4", out="bf16"),
        # one token, weights in 16 bits
        dict(name="moe_token", op="moe", t=1, h=2048, i=1024, e=64, k=6, x="bf16", w="bf16"),
        # a small decoding batch, weights in 4 bits
        dict(name="moe_tokens_4bit", op="moe", t=16, h=4096, i=1280, e=64, k=4, x="bf16", w="mx4"),
        # odd extents, as small models and tests have them
        dict(name="moe_ragged", op="moe", t=7, h=1000, i=333, e=10, k=3, x="f16", w="f16"),
        # a full decoding batch that reaches nearly every expert
        dict(name="moe_batch", op="moe", t=64, h=2048, i=1024, e=128, k=8, x="bf16", w="bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def _extent(rng, low, high):
    """Half of the extents are multiples of 64, as models have them, half are any."""
    n = _log(rng, low, high)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["round_trip", "product", "product", "moe", "moe"])
    while True:
        if op == "round_trip":
            c = dict(op=op, l=_log(rng, 1, 16), r=_log(rng, 1, 16384), c=_extent(rng, 1, 16384),
                     axis=rng.choice([-1, -2]), dtype=rng.choice(["f32", "bf16", "f16"]))
            if c["l"] * c["r"] * c["c"] <= MAX_ELEMENTS:
                return c
        elif op == "product":
            c = dict(op=op, l=rng.choice([1, 1, 2, 5, 16]), m=_log(rng, 1, 8192), n=_extent(rng, 16, 16384),
                     k=_extent(rng, 32, 16384), a=rng.choice(["f32", "bf16", "f16", "mx4"]),
                     b=rng.choice(["mx4", "mx4", "f32", "bf16"]), out=rng.choice(["f32", "bf16", "f16"]))
            operands = c["l"] * c["k"] * (c["m"] + c["n"])
            if c["l"] * c["m"] * c["n"] * c["k"] <= MAX_PRODUCT and operands <= MAX_ELEMENTS * 2 \
                    and c["l"] * c["m"] * c["n"] <= MAX_OUTPUT:
                return c
        else:
            e = _log(rng, 2, 128)
            x = rng.choice(["bf16", "f16"])
            c = dict(op=op, t=_log(rng, 1, 64), h=_extent(rng, 64, 8192), i=_extent(rng, 32, 8192), e=e,
                     k=rng.randint(1, min(e, 8)), x=x, w=rng.choice([x, "mx4"]))
            if c["e"] * 3 * c["h"] * c["i"] <= MAX_EXPERT_WEIGHTS:
                return c


def _mx4_blocks(x):
    """Codes uint8 [..., rows, ceil(k/32)*16] (two to a byte, the even index in
    the low half) and scale bytes [..., rows, ceil(k/32)] of x [..., rows, k]."""
    rows, k = x.shape[-2], x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)                           # top = f * 2^e, f in [0.5, 1)
    e = torch.where(top > 0, (e - 3).clamp(-127, 127), torch.full_like(e, -127))
    q = torch.ldexp(x, -e)
    code = _code_of(q)
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2)
    return codes.contiguous(), (e + 127).squeeze(-1).to(torch.uint8).contiguous()


def _code_of(q):
    m = q.abs()
    code = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    return code + (q < 0).to(torch.uint8) * 8


def _mx4_values(codes, scales, k, dtype=torch.float32):
    """The values [..., rows, k] that codes and scales stand for."""
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), dtype=dtype, device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = table[code.int()].unflatten(-1, (-1, 32))
    e = scales.to(torch.int32).unsqueeze(-1) - 127
    return torch.ldexp(v, e).flatten(-2)[..., :k]


def _mx4_rounded(x):
    """x [..., rows, k] replaced by the values of its 4-bit form."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -k % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)
    e = torch.where(top > 0, (e - 3).clamp(-127, 127), torch.full_like(e, -127))
    code = _code_of(torch.ldexp(x, -e))
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), device=x.device)
    return torch.ldexp(table[code.int()], e).flatten(-2)[..., :k]


def _activations(gen, shape, dtype):
    """Normal values with a few features ten times as large, as activations have them."""
    x = torch.randn(shape, generator=gen, device="cuda")
    wide = torch.rand(shape[-1], generator=gen, device="cuda") < 0.004
    return torch.where(wide, x * 10, x).to(DTYPES[dtype])


def _weights(gen, shape):
    return torch.randn(shape, generator=gen, device="cuda") * shape[-1] ** -0.5


class _Kept:
    """A matrix kept in 4 bits: codes and scales, and this package's form of them."""

    def __init__(self, x, k):
        self.k = k
        self.codes, self.scales = _mx4_blocks(x)
        if own:
            from custom_matmul_kernels_amd import MX4Tensor
            self.mx4 = MX4Tensor.from_blocks(self.codes, self.scales, k)

    def values(self, index=None):
        if index is None:
            return _mx4_values(self.codes, self.scales, self.k)
        return _mx4_values(self.codes[index], self.scales[index], self.k)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    if c["op"] == "round_trip":
        return {"case": c, "x": _activations(gen, (c["l"], c["r"], c["c"]), c["dtype"])}
    if c["op"] == "product":
        A = _activations(gen, (c["l"], c["m"], c["k"]), "f32" if c["a"] == "mx4" else c["a"])
        B = _weights(gen, (c["l"], c["n"], c["k"]))              # stored [n, k]
        A = _Kept(A, c["k"]) if c["a"] == "mx4" else A
        B = _Kept(B, c["k"]) if c["b"] == "mx4" else B.to(DTYPES[c["b"]])
        state = {"case": c, "A": A, "B": B}
        if own:
            from custom_matmul_kernels_amd import MX4BMMCUDA
            state["product"] = MX4BMMCUDA(out_dtype=DTYPES[c["out"]])
        return state
    x = _activations(gen, (c["t"], c["h"]), c["x"])
    router = _weights(gen, (c["e"], c["h"])).to(DTYPES[c["x"]])
    gate_up = _weights(gen, (c["e"], 2 * c["i"], c["h"]))
    gate_up = _Kept(gate_up, c["h"]) if c["w"] == "mx4" else gate_up.to(DTYPES[c["w"]])
    down = _weights(gen, (c["e"], c["h"], c["i"]))
    down = _Kept(down, c["i"]) if c["w"] == "mx4" else down.to(DTYPES[c["w"]])
    state = {"case": c, "x": x, "router": router, "gate_up": gate_up, "down": down}
    if own:
        from custom_matmul_kernels_amd import MoECUDA
        state["layer"] = MoECUDA(k=c["k"])
    return state


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    c = s["case"]
    if c["op"] == "round_trip":
        from custom_matmul_kernels_amd import quantize_mx4
        return quantize_mx4(s["x"], dim=c["axis"]).dequantize(DTYPES[c["dtype"]])
    if c["op"] == "product":
        A = s["A"].mx4 if c["a"] == "mx4" else s["A"]
        B = s["B"].mx4 if c["b"] == "mx4" else s["B"]
        return s["product"](A, B.transpose(1, 2))
    gate_up = s["gate_up"].mx4 if c["w"] == "mx4" else s["gate_up"]
    down = s["down"].mx4 if c["w"] == "mx4" else s["down"]
    return s["layer"](s["x"], s["router"], gate_up, down)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "round_trip":
        x = s["x"]
        if c["axis"] == -2:
            return _mx4_rounded(x.transpose(1, 2)).transpose(1, 2).to(x.dtype).contiguous()
        return _mx4_rounded(x).to(x.dtype).contiguous()
    if c["op"] == "product":
        A = s["A"].values() if c["a"] == "mx4" else _mx4_rounded(s["A"])
        B = s["B"].values() if c["b"] == "mx4" else _mx4_rounded(s["B"])
        return torch.matmul(A, B.transpose(1, 2)).to(DTYPES[c["out"]])
    x = s["x"].float()
    # 64-bit sums: two experts' scores may be close, and the choice must not hang on rounding
    score = torch.matmul(s["x"].double(), s["router"].double().t())
    order = torch.sort(score, dim=1, descending=True, stable=True)
    experts = order.indices[:, :c["k"]].contiguous()
    weights = torch.softmax(order.values[:, :c["k"]].float(), 1)
    kept = c["w"] == "mx4"
    if c["t"] * c["k"] <= c["e"]:                     # few choices: their weights alone
        i = experts.flatten()
        gate_up = s["gate_up"].values(i) if kept else s["gate_up"][i].float()
        down = s["down"].values(i) if kept else s["down"][i].float()
        u = torch.matmul(gate_up, x.repeat_interleave(c["k"], 0).unsqueeze(2)).squeeze(2)
        a = torch.nn.functional.silu(u[:, :c["i"]]) * u[:, c["i"]:]
        y = torch.matmul(down, a.unsqueeze(2)).squeeze(2).unflatten(0, (c["t"], c["k"]))
        y = (weights.unsqueeze(2) * y).sum(1)
    else:                                             # every expert for every token
        gate_up = s["gate_up"].values() if kept else s["gate_up"].float()
        down = s["down"].values() if kept else s["down"].float()
        u = torch.matmul(x.unsqueeze(0), gate_up.transpose(1, 2))
        a = torch.nn.functional.silu(u[..., :c["i"]]) * u[..., c["i"]:]
        y = torch.matmul(a, down.transpose(1, 2))     # [e, t, h]
        w = torch.zeros(c["t"], c["e"], device=x.device).scatter_(1, experts, weights)
        y = (w.t().unsqueeze(2) * y).sum(0)
    return y.to(s["x"].dtype), weights, experts


def work(case):
    c = case
    if c["op"] == "round_trip":
        n = c["l"] * c["r"] * c["c"]
        return {"bytes": 2 * n * SIZE[c["dtype"]], "flops": 2 * n}
    if c["op"] == "product":
        size = dict(SIZE, mx4=MX4_BYTES)
        b = c["l"] * (c["m"] * c["k"] * size[c["a"]] + c["n"] * c["k"] * size[c["b"]] + c["m"] * c["n"] * SIZE[c["out"]])
        return {"bytes": int(b), "flops": 2 * c["l"] * c["m"] * c["n"] * c["k"]}
    # the experts that a uniform choice of k for each token reaches
    reached = c["e"] * (1 - (1 - c["k"] / c["e"]) ** c["t"])
    weight = MX4_BYTES if c["w"] == "mx4" else SIZE[c["w"]]
    b = reached * 3 * c["h"] * c["i"] * weight + c["e"] * c["h"] * SIZE[c["x"]] \
        + 2 * c["t"] * c["h"] * SIZE[c["x"]] + c["t"] * c["k"] * 12
    return {"bytes": int(b), "flops": 2 * c["t"] * (c["k"] * 3 * c["h"] * c["i"] + c["e"] * c["h"])}


def _exact_rounded(x):
    """The 4-bit form's values in 64 bits, from its definition: the nearest of the
    sixteen values by distance, the even code where two are as near."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -k % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** -140)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)               # log2 may round up to a power of two
    unit = torch.exp2((e - 2).clamp_min(-127.0))
    q = (x / unit).abs().clamp_max(6.0)
    # magnitudes are evenly spaced by .5 up to 2, by 1 up to 4, by 2 up to 6; torch.round goes to even
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0)).to(q.dtype)
    v = torch.round(q / step) * step
    return (v * torch.sign(x) * unit).flatten(-2)[..., :k]


def _exact_values(kept, index=None):
    codes, scales = (kept.codes, kept.scales) if index is None else (kept.codes[index], kept.scales[index])
    code = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    m, e = code % 2, code // 2 % 4                               # mantissa bit, exponent bits
    v = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.exp2(e.double() - 1))
    v = torch.where(code >= 8, -v, v).unflatten(-1, (-1, 32))
    return (v * torch.exp2(scales.double() - 127).unsqueeze(-1)).flatten(-2)[..., :kept.k]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "round_trip":
        if c["axis"] == -2:
            return _exact_rounded(s["x"].transpose(1, 2)).transpose(1, 2).contiguous()
        return _exact_rounded(s["x"])
    if c["op"] == "product":
        A = _exact_values(s["A"]) if c["a"] == "mx4" else _exact_rounded(s["A"])
        B = _exact_values(s["B"]) if c["b"] == "mx4" else _exact_rounded(s["B"])
        return torch.bmm(A, B.transpose(1, 2).contiguous())
    x = s["x"].double()
    score = (x.unsqueeze(1) * s["router"].double()).sum(2)
    experts = score.argsort(dim=1, descending=True, stable=True)[:, :c["k"]].contiguous()
    picked = score.gather(1, experts)
    weights = torch.exp(picked - picked[:, :1])
    weights = weights / weights.sum(1, keepdim=True)
    y = torch.zeros(c["t"], c["h"], dtype=torch.float64, device=x.device)
    for e in experts.unique().tolist():
        one = slice(e, e + 1)
        gate_up = (_exact_values(s["gate_up"], one) if c["w"] == "mx4" else s["gate_up"][one].double())[0]
        down = (_exact_values(s["down"], one) if c["w"] == "mx4" else s["down"][one].double())[0]
        t, j = (experts == e).nonzero(as_tuple=True)
        u = x[t] @ gate_up.t()
        g, v = u[:, :c["i"]], u[:, c["i"]:]
        y[t] += weights[t, j].unsqueeze(1) * ((g / (1 + torch.exp(-g)) * v) @ down.t())
    return y, weights, experts
