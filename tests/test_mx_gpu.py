"""Microscaled 4-bit floating point (`mx_quantize`, `mx_dequantize`, `mx_gemm`, `mx_grouped_gemm`) against the format's
definition in 64 bits.

Quantisation is exact by its definition: bits are compared. Products: with scales of 1/2, 1 and 2 every term is a multiple
of 2^-4 below 2^8, so that sums of up to 4096 terms fit into the 24 bits of fp32 and have to come out exactly, whatever
their order. With scales of any size a sum of K terms in fp32, by adders that round or cut, is off by at most
K 2^-23 sum|term|; the rounding to the output's type adds eps / 2 of the value."""
import functools

import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# every kernel and tile: the library's choice, the few-token kernel, single CTAs, CTA pairs
TILES = [None] + [{"block_n": b} for b in (16, 32, 64)] + [{"block_n": b, "cta_group": 1} for b in (64, 128)] \
    + [{"block_n": b, "cta_group": 2} for b in (64, 128, 192, 256)]


def _values(data, scales):
    """Packed values and scales as 64-bit numbers."""
    data, scales = data.cpu(), scales.cpu().double()
    code = torch.stack((data & 15, data >> 4), -1).view(*data.shape[:-1], -1).long()
    v = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales - 127))
    return v * s.repeat_interleave(32, -1)


def _quantised64(x):
    """(packed values, scales) of x by the definition, the nearest of eight magnitudes, ties to the even code."""
    x = x.detach().cpu().double()
    b = x.reshape(-1, 32)
    bad = ~b.isfinite().all(1)
    most = b.abs().amax(1)
    e = torch.frexp(torch.where(bad | (most == 0), torch.ones_like(most), most)).exponent - 1 - 2
    e = torch.where(most == 0, -127, e.clamp_min(-127))
    a = torch.where(bad[:, None], torch.zeros_like(b), b / torch.exp2(e.double())[:, None])
    mid = (GRID[1:] + GRID[:-1]) / 2
    code = torch.zeros_like(a, dtype=torch.int64)
    for c in range(7):
        code += (a.abs() >= mid[c]) if c % 2 else (a.abs() > mid[c])
    code += 8 * torch.signbit(a)
    code[bad] = 0
    code = code.view(*x.shape).to(torch.uint8)
    scales = torch.where(bad, 255, e + 127).view(*x.shape[:-1], -1).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _random_mx(shape, seed, low=126, high=128):
    """Random codes with scales between two bytes."""
    import flux_b200 as flux

    g = torch.Generator().manual_seed(seed)
    data = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(low, high + 1, (*shape[:-1], shape[-1] // 32), generator=g, dtype=torch.uint8)
    return flux.MXTensor(data.cuda(), scales.cuda()), _values(data, scales)


def _status():
    import flux_b200 as flux

    torch.cuda.synchronize()
    flux.get_comm(None).check_status()


# ---------------------------------------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 96), (7, 544), (130, 1024), (1001, 160)])
def test_quantize_is_the_definition(rows, k, dtype):
    import flux_b200 as flux

    g = torch.Generator().manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(3 * torch.randn(rows, k // 32, generator=g)).repeat_interleave(32, 1)).to(dtype)
    q = flux.mx_quantize(x.cuda())
    data, scales = _quantised64(x)
    assert q.shape == (rows, k) and tuple(q.data.shape) == (rows, k // 2) and tuple(q.scales.shape) == (rows, k // 32)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.data.cpu(), data)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got, want = q.dequantize(out).cpu(), _values(data, scales).to(out)
        # (a block that overflowed fp16 before it came here is NaN)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])


def test_quantize_at_every_border():
    """All ties and their neighbours, both signs, at the ends of fp32's range and in between; zeros; what is no number."""
    import flux_b200 as flux

    marks = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995], dtype=torch.float32)
    near = torch.cat((marks, torch.nextafter(marks, torch.tensor(0.0)), torch.nextafter(marks, torch.tensor(8.0))))
    block = torch.cat((near, torch.tensor([4.0, 0.0])))
    signs = torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0)
    rows = [block * signs * 2.0 ** e for e in (0, 1, -1, 100, 125, -100, -120, -124, -126, -127, -140, -149)]
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), torch.finfo(torch.float32).max)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = block.clone()
        r[5] = bad
        rows.append(r)
    x = torch.stack(rows).float()
    q = flux.mx_quantize(x.cuda())
    data, scales = _quantised64(x)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.data.cpu(), data)
    got, want = q.dequantize(torch.float32).cpu(), _values(data, scales).to(torch.float32)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_quantize_layouts():
    """Strided rows, columns that are not contiguous, addresses between the vectors' boundaries, three dimensions."""
    import flux_b200 as flux

    g = torch.Generator().manual_seed(2)
    big = torch.randn(40, 200, generator=g).to(torch.bfloat16).cuda()
    views = [torch.randn(2, 130, 160, generator=g).cuda(), torch.randn(2, 3, 7, 32, generator=g).cuda().half(), big[:, 8:104], big[:, 3:131], big[::3, :64], big[:, ::2][:, :96], big.t()[:, :32], big[:1, :32].expand(5, 32),
             big.reshape(-1)[1:32 * 64 + 1].view(32, 64), torch.randn(3, 5, 64, generator=g).cuda()]
    for x in views:
        q = flux.mx_quantize(x)
        data, scales = _quantised64(x)
        assert torch.equal(q.data.cpu(), data) and torch.equal(q.scales.cpu(), scales)


def test_quantize_matrices_of_one_row():
    """Contiguous by torch's rules whatever the stride along the row that there is one of."""
    import flux_b200 as flux

    g = torch.Generator().manual_seed(8)
    for x in (torch.randn(3, 64, 1, generator=g).transpose(1, 2), torch.randn(2, 3, 96, 1, generator=g).transpose(2, 3),
              torch.randn(64, 1, generator=g).t(), torch.randn(5, 64, generator=g)[:, None, :]):
        x = x.cuda()
        q = flux.mx_quantize(x)
        data, scales = _quantised64(x)
        assert q.shape == x.shape and torch.equal(q.data.cpu(), data) and torch.equal(q.scales.cpu(), scales)


def test_quantize_into_the_order_of_experts():
    import flux_b200 as flux

    g = torch.Generator().manual_seed(3)
    for ntokens, topk, k in ((1, 1, 32), (33, 2, 544), (200, 5, 96)):
        chosen = torch.rand(ntokens, 8, generator=g).topk(topk, dim=1).indices.to(torch.int32)
        chosen[torch.rand(ntokens, topk, generator=g) < 0.2] = -1
        si, splits = flux.calc_scatter_index(chosen.cuda(), torch.empty(8), return_splits=True)
        x = torch.randn(ntokens, k, generator=g).to(torch.float16).cuda()
        whole, q = flux.mx_quantize(x), flux.mx_quantize(x, splits, si)
        assert torch.equal(q.data, flux.moe_permute(whole.data, splits, si))
        assert torch.equal(q.scales, flux.moe_permute(whole.scales.contiguous(), splits, si))


def test_dequantize_every_code_and_scale():
    import flux_b200 as flux

    data = (torch.arange(256 * 16) % 256).to(torch.uint8).view(256, 16)
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(256, 1)
    q = flux.MXTensor(data.cuda(), scales.cuda())
    want = _values(data, scales)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = q.dequantize(out).cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0, 9.0, -9.0), want.to(out).nan_to_num(0.0, 9.0, -9.0))


# -------------------------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("tuning", TILES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (16, 128, 256), (5, 130, 288), (100, 257, 2080), (225, 513, 544), (300, 1000, 4096), (1500, 2100, 1056)])
def test_product_is_exact(m, n, k, tuning):
    import flux_b200 as flux

    x, xv = _random_mx((m, k), m + k)
    w, wv = _random_mx((n, k), n + k + 1)
    if tuning in ({"block_n": 16}, {"block_n": 32}) and m > tuning["block_n"]:
        with pytest.raises(RuntimeError, match="is for up to"):
            flux.mx_gemm(x, w, output_dtype=torch.float32, tuning=tuning)
        return
    y = flux.mx_gemm(x, w, output_dtype=torch.float32, tuning=tuning)
    _status()
    assert torch.equal(y.cpu().double(), xv @ wv.t())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,bias", [(1, 3584, 8192, False), (48, 1031, 1024, True), (130, 96, 12288, True), (1000, 3588, 512, True)])
def test_product_of_quantised_matrices(m, n, k, bias, dtype):
    import flux_b200 as flux

    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * 0.02
    b = (torch.randn(n, generator=g) * 0.1).to(dtype) if bias else None
    xq, wq = flux.mx_quantize(x.to(torch.bfloat16).cuda()), flux.mx_quantize(w.to(torch.bfloat16).cuda())
    y = flux.mx_gemm(xq, wq, bias=None if b is None else b.cuda(), output_dtype=dtype)
    _status()
    xv, wv = _values(xq.data, xq.scales), _values(wq.data, wq.scales)
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias:
        want, size = want + b.double(), size + b.double().abs()
    off = k * 2.0 ** -23 * size
    off = off + torch.finfo(dtype).eps / 2 * (want.abs() + off)
    assert bool(((y.cpu().double() - want).abs() <= off).all())


def _grouped_want(xv, wv, splits):
    parts, r = [], 0
    for e, n in enumerate(splits):
        parts.append(xv[r:r + n] @ wv[e].t())
        r += n
    return torch.cat(parts)


@pytest.mark.parametrize("tuning", TILES, ids=str)
@pytest.mark.parametrize("splits,n,k", [([3], 128, 256), ([0, 5, 0, 1, 40, 0], 130, 288), ([17, 300, 0, 64, 1, 33, 224], 257, 544),
                                        ([1] * 100, 48, 96), ([0] * 40 + [200] + [0] * 300 + [7, 0], 70, 320), ([0, 0], 64, 64)])
def test_grouped_product_is_exact(splits, n, k, tuning):
    import flux_b200 as flux

    rows = sum(splits) + 9  # rows behind the last expert's: left as they were
    x, xv = _random_mx((rows, k), rows)
    w, wv = _random_mx((len(splits), n, k), n)
    out = torch.full((rows, n), -77.0, device="cuda")
    flux.mx_grouped_gemm(x, w, torch.tensor(splits, dtype=torch.int32, device="cuda"), torch.float32, output=out, tuning=tuning)
    _status()
    got = out.cpu().double()
    assert torch.equal(got[:sum(splits)], _grouped_want(xv, wv, splits))
    assert bool((got[sum(splits):] == -77.0).all())


def test_splits_that_do_not_fit_touch_nothing_outside():
    import flux_b200 as flux

    x, xv = _random_mx((50, 256), 1)
    w, wv = _random_mx((4, 64, 256), 2)
    for tuning in (None, {"block_n": 64, "cta_group": 2}):
        for splits, real in (([20, 100, 5, 5], [20, 30, 0, 0]), ([-5, 20, -1, 2 ** 31 - 1], [0, 20, 0, 30]), ([2 ** 31 - 1] * 4, [50, 0, 0, 0])):
            guard = torch.full((60, 64), -77.0, device="cuda")
            flux.mx_grouped_gemm(x, w, torch.tensor(splits, dtype=torch.int32, device="cuda"), torch.float32, output=guard[:50], tuning=tuning)
            _status()
            assert torch.equal(guard[:50].cpu().double(), _grouped_want(xv, wv, real))
            assert bool((guard[50:] == -77.0).all())


def test_nan_stays_in_its_row():
    """A block with the scale 255 makes its row (or column) of the result NaN and no other; scales at the ends of the range."""
    import flux_b200 as flux

    for tuning in (None, {"block_n": 64, "cta_group": 2}):
        for k in (64, 544):
            g = torch.Generator().manual_seed(k)
            data = torch.randint(0, 256, (20, k // 2), generator=g, dtype=torch.uint8)
            scales = torch.full((20, k // 32), 127, dtype=torch.uint8)
            scales[3, -1], scales[7, 0], scales[9, :], scales[11, :] = 255, 255, 0, 190
            x = flux.MXTensor(data.cuda(), scales.cuda())
            w, wv = _random_mx((40, k), 5)
            y = flux.mx_gemm(x, w, output_dtype=torch.float32, tuning=tuning).cpu().double()
            _status()
            bad = torch.zeros(20, dtype=torch.bool)
            bad[3] = bad[7] = True
            assert bool(y[bad].isnan().all()) and not bool(y[~bad].isnan().any())
            want = _values(data, scales)[~bad] @ wv.t()
            # row 9's terms are 2^-127 times multiples of 2^-4: fp32's subnormal steps hold them, rows of one scale are exact
            assert torch.equal(y[~bad], want)


def test_products_on_two_streams_and_in_graphs():
    import flux_b200 as flux

    x, xv = _random_mx((200, 2048), 1)
    w, wv = _random_mx((700, 2048), 2)
    few, fv = _random_mx((9, 2048), 3)
    splits = torch.tensor([150, 50], dtype=torch.int32, device="cuda")
    w2, w2v = _random_mx((2, 300, 2048), 4)
    want, want_few, want_g = xv @ wv.t(), fv @ wv.t(), _grouped_want(xv, w2v, [150, 50])
    f32 = torch.float32
    flux.mx_gemm(x, w, output_dtype=f32)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in (a, b):
            with torch.cuda.stream(s):
                outs.append((flux.mx_gemm(x, w, output_dtype=f32), flux.mx_gemm(few, w, output_dtype=f32), flux.mx_grouped_gemm(x, w2, splits, f32)))
    _status()
    for y, yf, yg in outs:
        assert torch.equal(y.cpu().double(), want) and torch.equal(yf.cpu().double(), want_few) and torch.equal(yg.cpu().double(), want_g)
    graphs, held = [], []
    tokens = torch.randn(64, 2048, device="cuda")
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            held.append((flux.mx_gemm(x, w, output_dtype=f32), flux.mx_gemm(flux.mx_quantize(tokens), w, output_dtype=f32),
                         flux.mx_grouped_gemm(x, w2, splits, f32)))
        graphs.append(g)
    tokens.normal_()
    splits.copy_(torch.tensor([30, 170], dtype=torch.int32))
    for s, g in zip((a, b), graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    _status()
    eager = flux.mx_gemm(flux.mx_quantize(tokens), w, output_dtype=f32)
    for y, yt, yg in held:
        assert torch.equal(y.cpu().double(), want) and torch.equal(yt, eager)
        assert torch.equal(yg.cpu().double(), _grouped_want(xv, w2v, [30, 170]))


def test_empty_operands_and_refusals():
    import flux_b200 as flux

    w = flux.mx_quantize(torch.randn(64, 96, device="cuda"))
    x = flux.mx_quantize(torch.empty(0, 96, device="cuda"))
    assert flux.mx_gemm(x, w).shape == (0, 64) and x.dequantize().shape == (0, 96)
    one = flux.mx_quantize(torch.randn(3, 96, device="cuda"))
    cases = [
        (lambda: flux.mx_quantize(torch.randn(4, 40, device="cuda")), "multiple of 32"),
        (lambda: flux.mx_quantize(torch.zeros(4, 64, dtype=torch.int32, device="cuda")), "fp32, bf16 or fp16"),
        (lambda: flux.mx_quantize(torch.randn(4, 64, device="cuda", requires_grad=True)), "no gradient"),
        (lambda: flux.mx_quantize(torch.randn(4, 64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")), "belong together"),
        (lambda: flux.mx_gemm(one, flux.mx_quantize(torch.randn(64, 64, device="cuda"))), "K 64 != input K 96"),
        (lambda: flux.mx_gemm(one, w, output_dtype=torch.int32), "output must be"),
        (lambda: flux.mx_gemm(one, w, bias=torch.zeros(64, device="cuda")), "bias"),
        (lambda: flux.mx_gemm(one, w, output=torch.empty(3, 63, dtype=torch.bfloat16, device="cuda")), "output has"),
        (lambda: flux.mx_gemm(one, w, tuning={"block_n": 48}), "block_n=48"),
        (lambda: flux.mx_gemm(one, w, tuning={"block_n": 64, "cta_group": 3}), "cta_group=3"),
        (lambda: flux.mx_grouped_gemm(one, w, torch.zeros(1, dtype=torch.int32, device="cuda")), "operands"),
        (lambda: flux.MXTensor(torch.zeros(4, 24, dtype=torch.uint8, device="cuda"), torch.zeros(4, 1, dtype=torch.uint8, device="cuda")), "multiple of 32"),
        (lambda: flux.MXTensor(torch.zeros(4, 16, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, dtype=torch.uint8, device="cuda")), "scales shape"),
    ]
    for call, words in cases:
        with pytest.raises(RuntimeError, match=words):
            call()


def test_a_bias_with_a_gradient_is_refused():
    import flux_b200 as flux

    x, w = (flux.mx_quantize(torch.randn(n, 96, device="cuda")) for n in (3, 64))
    bias = torch.zeros(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        flux.mx_gemm(x, w, bias=bias)
    with torch.no_grad():
        assert torch.equal(flux.mx_gemm(x, w, bias=bias), flux.mx_gemm(x, w))


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.parametrize("n,tuning", [(32768, None), (32771, None), (32768, {"block_n": 128, "cta_group": 1}), (32771, {"block_n": 64})], ids=str)
def test_products_of_more_than_31_bits_of_values(n, tuning):
    import flux_b200 as flux

    m, splits = 66000, [9000, 0, 20001, 36998]
    x, xv = _random_mx((m, 32), 1)
    w, wv = _random_mx((n, 32), 2)
    w3, w3v = _random_mx((4, n, 32), 3)
    y = flux.mx_gemm(x, w, tuning=tuning)
    _status()
    for r in (slice(0, 40), slice(m // 2, m // 2 + 40), slice(m - 40, m)):
        assert torch.equal(y[r].cpu(), (xv[r] @ wv.t()).to(torch.bfloat16))
    y = flux.mx_grouped_gemm(x, w3, torch.tensor(splits, dtype=torch.int32, device="cuda"), output=y, tuning=tuning)
    _status()
    for e, r in ((0, slice(0, 40)), (0, slice(8960, 9000)), (2, slice(9000, 9040)), (3, slice(m - 41, m - 1))):
        assert torch.equal(y[r].cpu(), (xv[r] @ w3v[e].t()).to(torch.bfloat16))
    assert torch.equal(y[-1].cpu(), (xv[-1] @ wv.t()).to(torch.bfloat16))  # the row past the last expert's is the one from before


def test_quantise_more_than_32_bits_of_values():
    import flux_b200 as flux

    rows, k = 540000, 8192
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    part = torch.randn(1000, k, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    for r in range(0, rows, 1000):
        torch.mul(part.cuda(), 1.0 + r / rows, out=x[r:r + 1000])
    q = flux.mx_quantize(x)
    y = q.dequantize()
    for r in (slice(0, 30), slice(rows // 2 + 7, rows // 2 + 40), slice(rows - 30, rows)):
        data, scales = _quantised64(x[r])
        assert torch.equal(q.data[r].cpu(), data)
        assert torch.equal(y[r].cpu().double(), _values(data, scales))


@pytest.mark.parametrize("lead", [(), (3,)])
def test_copies_outlive_what_they_were_copied_from(lead):
    import copy
    import io

    import flux_b200 as flux

    x, v = flux.mx_quantize(torch.randn(5, 96, device="cuda")), torch.randn(*lead, 40, 96, device="cuda")
    w = flux.mx_quantize(v)
    splits = torch.tensor([2, 1, 2], dtype=torch.int32, device="cuda")

    def product(q):
        return flux.mx_grouped_gemm(x, q, splits) if lead else flux.mx_gemm(x, q)

    want, values = product(w), w.dequantize()
    f = io.BytesIO()
    torch.save(w, f)
    f.seek(0)
    copies = [copy.deepcopy(w), copy.copy(w), torch.load(f, weights_only=False)]
    del w
    trash = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (8192, 16384, 65536) for _ in range(4)]  # where it was
    for c in copies:
        assert torch.equal(product(c), want) and torch.equal(c.dequantize(), values)
    del trash


# ------------------------------------------------------------------------------------ several tiles of several stages a CTA
PERSISTENT = [t for t in TILES if t and "cta_group" in t]


@functools.lru_cache(maxsize=64)
def _shared(shape, seed):
    """`_random_mx`, the values on the GPU: made once for all variants."""
    q, v = _random_mx(shape, seed)
    return q, v.cuda()


def _same(got, want):
    """Exact sums, rounded once to the type of `got`."""
    assert torch.equal(got, want.to(got.dtype))


@pytest.mark.parametrize("dtype,n", [(torch.float32, 600), (torch.bfloat16, 600), (torch.bfloat16, 601)])
@pytest.mark.parametrize("num_ctas", [2, 3, 6])
@pytest.mark.parametrize("tuning", PERSISTENT, ids=str)
def test_product_of_several_tiles_a_cta_is_exact(tuning, num_ctas, dtype, n):
    """Few CTAs take all tiles: accumulators, scale slots and stages go from tile to tile, with less than, about and more K than
    the ring and the slots hold."""
    import flux_b200 as flux

    m = 800
    for k in (96, 544, 1056, 2336):
        x, xv = _shared((m, k), m + k)
        w, wv = _shared((n, k), n + k + 1)
        y = flux.mx_gemm(x, w, output_dtype=dtype, tuning={**tuning, "num_ctas": num_ctas})
        _status()
        _same(y, xv @ wv.t())


@pytest.mark.parametrize("dtype,n", [(torch.float32, 520), (torch.bfloat16, 520), (torch.bfloat16, 519)])
@pytest.mark.parametrize("num_ctas", [2, 3, 6])
@pytest.mark.parametrize("tuning", PERSISTENT, ids=str)
def test_grouped_product_of_several_tiles_a_cta_is_exact(tuning, num_ctas, dtype, n):
    import flux_b200 as flux

    splits = [300, 0, 517, 64, 1, 130, 257, 0, 3]
    rows = sum(splits) + 5
    for k in (96, 544, 1312, 2336):
        x, xv = _shared((rows, k), rows + k)
        w, wv = _shared((len(splits), n, k), n + k)
        out = torch.full((rows, n), -77.0, device="cuda", dtype=dtype)
        flux.mx_grouped_gemm(x, w, torch.tensor(splits, dtype=torch.int32, device="cuda"), dtype, output=out, tuning={**tuning, "num_ctas": num_ctas})
        _status()
        _same(out[:-5], _grouped_want(xv, wv, splits))
        assert bool((out[-5:] == -77.0).all())


@pytest.mark.parametrize("tuning", [None, *PERSISTENT], ids=str)
def test_products_of_several_waves_are_exact(tuning):
    """Every SM takes several tiles."""
    import flux_b200 as flux

    k = 1056
    x, xv = _shared((4100, k), 1)
    w, wv = _shared((8200, k), 2)
    y = flux.mx_gemm(x, w, output_dtype=torch.bfloat16, tuning=tuning)
    _status()
    _same(y, xv @ wv.t())
    splits = [900, 17, 0, 2050, 333, 800]
    w, wv = _shared((6, 4104, k), 3)
    y = flux.mx_grouped_gemm(x, w, torch.tensor(splits, dtype=torch.int32, device="cuda"), tuning=tuning)
    _status()
    _same(y, _grouped_want(xv, wv, splits))


@pytest.mark.parametrize("dtype,exponents", [(torch.bfloat16, (0, 1, -1, 100, 125, -100, -119, -120, -124, -125, -126, -127, -129, -132)),
                                             (torch.float16, (0, 1, -1, 12, 13, -8, -11, -13, -14, -16, -19, -23))])
def test_quantize_at_every_border_of_16_bits(dtype, exponents):
    """All ties and their neighbours in the input's own type, at the ends of its range, among its subnormal numbers, and in between."""
    import flux_b200 as flux

    marks = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9], dtype=dtype)
    bits = marks.view(torch.int16)
    near = torch.cat((marks, (bits - 1).view(dtype), (bits + 1).view(dtype)))
    block = torch.cat((near, torch.tensor([4.0, 0.0], dtype=dtype))).float()
    signs = torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0)
    rows = [block * signs * 2.0 ** e for e in exponents]
    # neighbours whose last bits the scaling by 2^e pushed out come back: the smallest numbers of the type, all of them
    small = torch.arange(32 * 64, dtype=torch.int16).view(dtype).view(-1, 32).float()
    rows += [*small, *(-small.flip(1))]
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), torch.finfo(dtype).max), torch.full((32,), torch.finfo(dtype).smallest_normal)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = block.clone()
        r[5] = bad
        rows.append(r)
    x = torch.stack(rows).to(dtype)
    data, scales = _quantised64(x)
    q = flux.mx_quantize(x.cuda())
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.data.cpu(), data)
    got, want = q.dequantize(torch.float32).cpu(), _values(data, scales).to(torch.float32)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    # unaligned rows go by another way to the same values
    wide = torch.zeros(x.shape[0], 67, dtype=dtype, device="cuda")
    wide[:, 3:35] = x.cuda()
    again = flux.mx_quantize(wide[:, 3:35])
    assert torch.equal(again.data, q.data) and torch.equal(again.scales, q.scales)


def test_quantise_more_rows_than_a_launch_takes():
    """Units of 16 (and back, of 8) values are numbered in 31 bits, 8 (4) for a row of 32 here: three launches and two."""
    import flux_b200 as flux

    torch.cuda.empty_cache()
    rows, part_rows = 537_000_000, 1_000_000
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    x = torch.empty(rows // part_rows, part_rows, 32, dtype=torch.bfloat16, device="cuda")
    part = torch.randn(part_rows, 32, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    for i in range(x.shape[0]):
        torch.mul(part, 1.0 + i / x.shape[0], out=x[i])
    x = x.view(rows, 32)
    q = flux.mx_quantize(x)
    y = q.dequantize()
    block_rows = 128
    for first in (0, 268_435_327, 2 * 268_435_327, 536_870_655, rows - 20):  # launches of the quantisation, and back, begin there
        r = slice(max(first - 20, 0), min(first + 20, rows))
        data, scales = _quantised64(x[r])
        assert torch.equal(q.data[r].cpu(), data)
        assert torch.equal(y[r].cpu().double(), _values(data, scales))
        b0 = r.start // block_rows
        some = q.blocks[b0:(r.stop - 1) // block_rows + 1].view(-1, 1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, 4)
        assert torch.equal(some[r.start - b0 * block_rows:r.stop - b0 * block_rows, :1].cpu(), scales)
        assert not bool(some[r.start - b0 * block_rows:r.stop - b0 * block_rows, 1:].any())
    del x, y, q
    torch.cuda.empty_cache()
