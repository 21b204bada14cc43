"""The operators that a mixture-of-experts layer with microscaled 4-bit weights is made of, and what they are timed on.

Every case is a call, or the short chain of calls, that a layer makes through the public entry points of `flux_b200`,
beside the same operator in its plain form (elementary torch operations in 32 bits, rounded once at the end):

  route    `moe_route`: the experts of every token and their weights from the router's logits; with its gradient
  sort     `moe_permute` and `moe_unpermute`: tokens in the order of their experts and back, with the routing weights
           applied; with all gradients
  quant    `mx_quantize` and back: 4-bit values (e2m1) with one power of two for every 32 of them
  product  `mx_quantize` of the tokens and `mx_gemm` with weights that were quantised when they were loaded
  grouped  `mx_quantize` of the tokens into the order of their experts and `mx_grouped_gemm`: a MoE layer's up projection

Sizes are shares of the layers that the benchmark and the tests name (hidden 4096, 8192, 12288; ffn 14336, 28672,
49152; 8 experts top-2, 32 experts top-4), and sizes between them. Activations are N(0, 1) with channels of unequal
size, weights N(0, 0.02), routing logits N(0, 1).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32  # values that share a scale


def listed():
    return [
        # the routing of one decoded batch: a call that costs more than its arithmetic
        {"name": "route_decode", "kind": "route", "dtype": "fp32", "tokens": 64, "experts": 8, "topk": 2, "train": False},
        # a training batch over many small experts, with the gradient of the logits
        {"name": "route_train", "kind": "route", "dtype": "bf16", "tokens": 16384, "experts": 64, "topk": 6, "train": True},
        # a few decoded sequences
        {"name": "sort_decode", "kind": "sort", "dtype": "bf16", "tokens": 7, "hidden": 4096, "experts": 8, "topk": 2, "drop": 0.0, "train": False},
        # a ragged chunk of a prompt with padding tokens, an odd hidden size
        {"name": "sort_ragged", "kind": "sort", "dtype": "fp16", "tokens": 2000, "hidden": 5124, "experts": 32, "topk": 4, "drop": 0.1, "train": False},
        # the benchmark's MoE batch, forward and backward
        {"name": "sort_train", "kind": "sort", "dtype": "bf16", "tokens": 8192, "hidden": 4096, "experts": 8, "topk": 2, "drop": 0.0, "train": True},
        # the activations of one decoded batch
        {"name": "quant_tokens", "kind": "quant", "dtype": "fp16", "rows": 48, "k": 12288},
        # a quarter of one layer's weights when they are loaded
        {"name": "quant_weights", "kind": "quant", "dtype": "bf16", "rows": 14336, "k": 12288},
        # decoding one sequence (an eighth of hidden 8192, ffn 28672)
        {"name": "product_decode", "kind": "product", "dtype": "bf16", "m": 1, "n": 3584, "k": 8192, "bias": False},
        # a ragged chunk of a prompt with a bias (a quarter of hidden 4096, ffn 14336)
        {"name": "product_ragged", "kind": "product", "dtype": "fp16", "m": 1000, "n": 3588, "k": 4096, "bias": True},
        # a prefill batch through an undivided projection: the benchmark's quantised configuration
        {"name": "product_prefill", "kind": "product", "dtype": "bf16", "m": 8192, "n": 28672, "k": 8192, "bias": False},
        # decoding a batch: every expert's weights are read for a few tokens (a quarter of ffn 14336)
        {"name": "grouped_decode", "kind": "grouped", "dtype": "bf16", "tokens": 64, "hidden": 4096, "ffn": 3584, "experts": 8, "topk": 2},
        # the benchmark's MoE configuration
        {"name": "grouped_prefill", "kind": "grouped", "dtype": "bf16", "tokens": 8192, "hidden": 4096, "ffn": 14336, "experts": 8, "topk": 2},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(int(round(v / step)) * step, lo), hi))


def draw(rng):
    kind = rng.choice(["route", "sort", "sort", "quant", "product", "product", "product", "grouped", "grouped"])
    if kind == "quant":
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _log(rng, 1, 16384), "k": _log(rng, 32, 12288, BLOCK)}
    if kind == "product":
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "m": _log(rng, 1, 8192), "n": _log(rng, 128, 28672),
                "k": _log(rng, 256, 8192, BLOCK), "bias": rng.random() < 0.4}
    experts = _log(rng, 4, 128)
    topk = rng.randint(1, min(8, experts))
    if kind == "route":
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp32"]), "tokens": _log(rng, 1, 32768), "experts": experts, "topk": topk,
                "train": rng.random() < 0.5}
    if kind == "sort":
        # at most 8192 x 12288 values of rows
        tokens = _log(rng, 1, 8192)
        return {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "tokens": tokens,
                "hidden": _log(rng, 64, max(64, min(8192, 8192 * 12288 // (tokens * topk)))), "experts": experts, "topk": topk,
                "drop": rng.choice([0.0, 0.0, 0.2]), "train": rng.random() < 0.5}
    # at most 8 x 14336 x 4096 values of weights and 16384 rows
    hidden = _log(rng, 256, 8192, BLOCK)
    return {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "tokens": _log(rng, 1, max(1, 16384 // topk)), "hidden": hidden,
            "ffn": _log(rng, 128, max(128, min(14336, 8 * 14336 * 4096 // (experts * hidden)))), "experts": experts, "topk": topk}


# ------------------------------------------------------------------------------------------------ inputs
class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        t = torch.randn(shape, generator=self.g, device="cuda", dtype=dtype)
        return t if std == 1.0 else t.mul_(std)

    def activations(self, rows, cols, dtype):
        size = torch.exp(0.5 * torch.randn((cols,), generator=self.g, device="cuda"))
        return (torch.randn((rows, cols), generator=self.g, device="cuda") * size).to(dtype)

    def weights(self, rows, cols):
        """Quantised weights as a checkpoint holds them: two values a byte, low half first, and a byte for every 32."""
        data = torch.empty((rows, cols // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((rows, cols // BLOCK), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // cols)
        for r in range(0, rows, step):
            v, s = _quantise(self.normal(min(step, rows - r), cols, std=0.02))
            code = _codes(v)
            data[r:r + step] = code[:, 0::2] | (code[:, 1::2] << 4)
            scales[r:r + step] = s
        return data, scales

    def routing(self, tokens, experts, topk, drop):
        """Chosen experts (-1: none), the row of every pair in the order of the experts (-1), rows for each expert, weights."""
        logits = self.normal(tokens, experts)
        w, chosen = torch.topk(torch.softmax(logits, -1), topk, dim=-1)
        if drop:
            gone = torch.rand((tokens, topk), generator=self.g, device="cuda") < drop / 2
            gone |= torch.rand((tokens, 1), generator=self.g, device="cuda") < drop / 2  # padding: no expert at all
            chosen = chosen.masked_fill(gone, -1)
        flat = chosen.reshape(-1)
        key = torch.where(flat < 0, experts, flat)
        order = torch.argsort(key, stable=True)
        place = torch.empty_like(order)
        place[order] = torch.arange(order.numel(), device="cuda")
        index = torch.where(flat < 0, -1, place).to(torch.int32).view(tokens, topk)
        splits = torch.bincount(key, minlength=experts + 1)[:experts].to(torch.int32)
        return index, splits, (w / w.sum(-1, keepdim=True)).contiguous()


def prepare(case, seed):
    mk = _Maker(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    st = {"case": case}
    if kind == "route":
        st["logits"] = mk.normal(case["tokens"], case["experts"]).to(dt).requires_grad_(case["train"])
        st["dw"] = mk.normal(case["tokens"], case["topk"])
    elif kind == "sort":
        t, h, k = case["tokens"], case["hidden"], case["topk"]
        st["index"], st["splits"], st["w"] = mk.routing(t, case["experts"], k, case["drop"])
        st["x"], st["y"] = mk.normal(t, h, dtype=dt), mk.normal(t * k, h, dtype=dt)
        if case["train"]:
            for name in ("x", "y", "w"):
                st[name].requires_grad_(True)
            st["dx_rows"], st["dout"] = mk.normal(t * k, h, dtype=dt), mk.normal(t, h, dtype=dt)
    elif kind == "quant":
        st["x"] = mk.activations(case["rows"], case["k"], dt)
    elif kind == "product":
        st["x"] = mk.activations(case["m"], case["k"], dt)
        st["data"], st["scales"] = mk.weights(case["n"], case["k"])
        st["bias"] = mk.normal(case["n"], std=0.1).to(dt) if case["bias"] else None
    else:
        e, h, f = case["experts"], case["hidden"], case["ffn"]
        st["x"] = mk.activations(case["tokens"], h, dt)
        data, scales = mk.weights(e * f, h)
        st["data"], st["scales"] = data.view(e, f, -1), scales.view(e, f, -1)
        st["index"], st["splits"], _ = mk.routing(case["tokens"], e, case["topk"], 0.0)
        st["longest"] = int(st["splits"].max())
    if own and "data" in st:
        import flux_b200 as flux

        st["wq"] = flux.MXTensor(st["data"], st["scales"])
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """(values of e2m1, their blocks' exponents + 127): the exponent of a block's largest value less that of the largest
    e2m1 value, 4; rounded to nearest, ties to even, 6 at most. A block with an infinity or a NaN has the exponent 255."""
    rows, cols = x.shape
    x = x.float().view(rows, cols // BLOCK, BLOCK)
    field = x.abs().amax(-1).view(torch.int32) >> 23
    scale = torch.where(field == 255, 255, (field - 2).clamp_min(0))
    a = x * ((254 - scale.clamp_max(253)) << 23).view(torch.float32)[..., None]
    s = a.abs()
    step = torch.where(s < 2, 0.5, torch.where(s < 4, 1.0, 2.0))
    v = torch.copysign((torch.round(s / step) * step).clamp_max(6.0), a)
    return v.view(rows, cols), scale.to(torch.uint8)


def _codes(v):
    """e2m1 values as 4-bit codes: sign, two bits of exponent, one of mantissa."""
    s = v.abs()
    mag = torch.where(s < 2, s * 2, torch.where(s < 4, s + 2, s / 2 + 4))
    return (mag + 8.0 * torch.signbit(v)).to(torch.uint8)


def _scale_values(scales):
    s = scales.to(torch.int32)
    bits = torch.where(s == 0, 1 << 22, torch.where(s == 255, 0x7FC00000, s << 23))
    return bits.to(torch.int32).view(torch.float32)


def _fake_quantised(x):
    v, s = _quantise(x)
    return (v.view(*s.shape, BLOCK) * _scale_values(s)[..., None]).view(x.shape)


def _dequantised(data, scales):
    """The 32-bit values of packed weights."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=data.device)
    code = torch.stack((data & 15, data >> 4), dim=-1).view(*scales.shape, BLOCK)
    return (table[code.int()] * _scale_values(scales)[..., None]).view(*data.shape[:-1], data.shape[-1] * 2)


def _plain(st):
    case = st["case"]
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "route":
        z = st["logits"].detach().float()
        top, chosen = torch.sort(z, dim=1, descending=True, stable=True)
        top, chosen = top[:, :case["topk"]], chosen[:, :case["topk"]]
        w = torch.exp(top - top[:, :1])
        w = w / w.sum(1, keepdim=True)
        out = (chosen.to(torch.int32), w)
        if case["train"]:
            g = w * (st["dw"] - (w * st["dw"]).sum(1, keepdim=True))
            out += (torch.zeros_like(z).scatter(1, chosen, g).to(dt),)
        return out
    if kind == "sort":
        t, k = st["index"].shape
        rows = t * k
        index = torch.where(st["index"] < 0, rows, st["index"]).long().view(-1)  # pairs without an expert: a row of their own

        def permuted(x):
            return torch.zeros((rows + 1, x.shape[1]), dtype=x.dtype, device=x.device).index_copy(0, index, x.repeat_interleave(k, 0))[:rows]

        def gathered(y):
            return torch.cat((y, y.new_zeros((1, y.shape[1]))))[index].float().view(t, k, -1)

        x, y, w = st["x"].detach(), st["y"].detach(), st["w"].detach()
        g = gathered(y)
        out = (permuted(x), (g * w[..., None]).sum(1).to(dt))
        if case["train"]:
            dout = st["dout"].float()
            dx = gathered(st["dx_rows"]).sum(1).to(dt)
            spread = torch.zeros((rows + 1, y.shape[1]), dtype=dt, device=y.device)
            dy = spread.index_copy(0, index, (dout[:, None] * w[..., None]).to(dt).view(rows, -1))[:rows]
            out += (dx, dy, (g * dout[:, None]).sum(2))
        return out
    if kind == "quant":
        return _fake_quantised(st["x"]).to(torch.bfloat16)
    xq = _fake_quantised(st["x"])
    w = _dequantised(st["data"], st["scales"])
    if kind == "product":
        y = xq @ w.t()
        return (y if st["bias"] is None else y + st["bias"].float()).to(dt)
    # every expert's rows, padded to the longest run
    t, k = st["index"].shape
    source = torch.empty((t * k,), dtype=torch.int64, device=xq.device)
    source[st["index"].long().view(-1)] = torch.arange(t * k, device=xq.device) // k
    ends = torch.cumsum(st["splits"].long(), 0)
    slot = torch.arange(st["longest"], device=xq.device)
    row = (ends - st["splits"])[:, None] + slot
    padded = torch.bmm(xq[source[row.clamp_max(t * k - 1)]], w.transpose(1, 2))
    at = torch.arange(t * k, device=xq.device)
    expert = torch.searchsorted(ends, at, right=True)
    return padded[expert, at - (ends - st["splits"])[expert]].to(dt)


def run(st):
    if not own:
        return _plain(st)
    import flux_b200 as flux

    case = st["case"]
    kind = case["kind"]
    if kind == "route":
        chosen, w = flux.moe_route(st["logits"], case["topk"])
        if case["train"]:
            return (chosen, w.detach()) + torch.autograd.grad(w, st["logits"], st["dw"])
        return chosen, w
    if kind == "sort":
        rows = flux.moe_permute(st["x"], st["splits"], st["index"])
        out = flux.moe_unpermute(st["y"], st["splits"], st["index"], st["w"])
        if case["train"]:
            return (rows.detach(), out.detach()) + torch.autograd.grad((rows, out), (st["x"], st["y"], st["w"]), (st["dx_rows"], st["dout"]))
        return rows, out
    if kind == "quant":
        return flux.mx_dequantize(flux.mx_quantize(st["x"]), torch.bfloat16)
    dt = DTYPES[case["dtype"]]
    if kind == "product":
        return flux.mx_gemm(flux.mx_quantize(st["x"]), st["wq"], bias=st["bias"], output_dtype=dt)
    xq = flux.mx_quantize(st["x"], st["splits"], st["index"])
    return flux.mx_grouped_gemm(xq, st["wq"], st["splits"], output_dtype=dt)


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        return {"bytes": t * (e * size * (2 if case["train"] else 1) + k * (12 if case["train"] else 8)), "flops": t * (e + 8 * k)}
    if kind == "sort":
        t, h, k = case["tokens"], case["hidden"], case["topk"]
        rows, idx = t * k * (1.0 - case["drop"]), t * k * 8
        if not case["train"]:
            return {"bytes": (2 * t + 2 * rows) * h * size + idx, "flops": 2.0 * rows * h}
        return {"bytes": (4 * t + 4 * rows) * h * size + idx + t * k * 4, "flops": 6.0 * rows * h}
    if kind == "quant":
        return {"bytes": case["rows"] * case["k"] * (size + 2), "flops": 3.0 * case["rows"] * case["k"]}
    packed = 0.5 + 1.0 / BLOCK
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * size + n * k * packed + m * n * size, "flops": 2.0 * m * n * k}
    t, h, f, e, k = (case[x] for x in ("tokens", "hidden", "ffn", "experts", "topk"))
    used = e * (1.0 - (1.0 - k / e) ** t)  # experts that get at least one token, on average
    return {"bytes": used * f * h * packed + t * h * size + t * k * f * size, "flops": 2.0 * t * k * f * h}


# ------------------------------------------------------------------------------------------------ 64 bits
def _nearest64(x):
    """Microscaled values of x from the definition: the nearest of the eight magnitudes, ties to the even code."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    half = (grid[1:] + grid[:-1]) / 2
    odd = torch.arange(7, device=x.device) % 2 == 1  # a tie between codes c and c + 1 goes up where c is odd
    step = max(1, (1 << 24) // x.shape[1])
    for r in range(0, x.shape[0], step):
        b = x[r:r + step].double().view(-1, BLOCK)
        most = b.abs().amax(1, keepdim=True)
        e = (torch.frexp(most).exponent - 1 - 2).clamp_min(-127).double()
        e = torch.where(most == 0, -127.0, e)
        a = b * torch.exp2(-e)
        mag = a.abs()
        code = torch.zeros_like(mag, dtype=torch.int64)
        for c in range(7):
            code += torch.where(odd[c], mag >= half[c], mag > half[c])
        v = torch.where(a < 0, -grid[code], grid[code]) * torch.exp2(e)
        out[r:r + step] = v.view(-1, x.shape[1])
    return out


def _weights64(data, scales):
    lo, hi = (data & 15).long(), (data >> 4).long()
    both = torch.empty((*data.shape[:-1], data.shape[-1], 2), dtype=torch.float64, device=data.device)
    for i, c in enumerate((lo, hi)):
        ex, man = (c >> 1) & 3, c & 1
        mag = torch.where(ex == 0, 0.5 * man, torch.exp2(ex.double() - 1) * (1 + 0.5 * man))
        both[..., i] = torch.where(c >= 8, -mag, mag)
    return both.view(*data.shape[:-1], -1) * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _mm64(a, data, scales):
    """a @ weights.T in 64 bits, a block of the weights' rows at a time."""
    out = torch.empty((a.shape[0], data.shape[0]), dtype=torch.float64, device=a.device)
    step = max(1, (1 << 25) // a.shape[1])
    for r in range(0, data.shape[0], step):
        out[:, r:r + step] = a @ _weights64(data[r:r + step], scales[r:r + step]).t()
    return out


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        z = st["logits"].double()
        experts = torch.arange(z.shape[1], device=z.device)
        ahead = (z[:, None, :] > z[:, :, None]) | ((z[:, None, :] == z[:, :, None]) & (experts[None, :] < experts[:, None])[None]) \
            if z.shape[0] * z.shape[1] ** 2 < 1 << 28 else None
        if ahead is None:  # the same, a block of tokens at a time
            rank = torch.cat([((b[:, None, :] > b[:, :, None]) | ((b[:, None, :] == b[:, :, None]) & (experts[None, :] < experts[:, None])[None])).sum(2)
                              for b in z.split(1024)])
        else:
            rank = ahead.sum(2)
        chosen = torch.argsort(rank, dim=1)[:, :case["topk"]]
        w = torch.softmax(z.gather(1, chosen), dim=1)
        out = (chosen.to(torch.int32), w)
        if case["train"]:
            z = z.requires_grad_(True)
            with torch.enable_grad():
                p = torch.softmax(z.gather(1, chosen), dim=1)
            out += torch.autograd.grad(p, z, st["dw"].double())
        return out
    if kind == "sort":
        index = st["index"].long()
        t, k = index.shape
        h = case["hidden"]
        pair = (index.reshape(-1) >= 0).nonzero().view(-1)
        at, token, choice = index.reshape(-1)[pair], pair // k, pair % k
        x, y, w = st["x"].double(), st["y"].double(), st["w"].double()
        rows = torch.zeros((t * k, h), dtype=torch.float64, device=x.device)
        rows[at] = x[token]
        wp = w[token, choice][:, None]
        out = (rows, torch.zeros_like(x).index_add_(0, token, y[at] * wp))
        if case["train"]:
            dout, dw, dy = st["dout"].double(), torch.zeros_like(w), torch.zeros_like(rows)
            dw[token, choice] = (y[at] * dout[token]).sum(1)
            dy[at] = dout[token] * wp
            out += (torch.zeros_like(x).index_add_(0, token, st["dx_rows"].double()[at]), dy, dw)
        return out
    xq = _nearest64(st["x"])
    if kind == "quant":
        return xq
    if kind == "product":
        y = _mm64(xq, st["data"], st["scales"])
        return y if st["bias"] is None else y + st["bias"].double()
    t, k = st["index"].shape
    source = torch.argsort(st["index"].reshape(-1)) // k
    runs = torch.split(source, st["splits"].tolist())
    return torch.cat([_mm64(xq[s], st["data"][e], st["scales"][e]) for e, s in enumerate(runs)])
