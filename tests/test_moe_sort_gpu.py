"""The token side of a MoE layer (`moe_route`, `moe_permute`, `moe_unpermute`) against its definition in 64 bits.

Tolerances: u = 2^-24 is half a step of fp32, u_t = eps(t) / 2 that of the output type. A sum of n terms in fp32, in any
order, is off by at most n u sum|term|; a rounding to the output type adds u_t |value|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _within(got, want, bound):
    got = got.double().cpu()
    off = (got - want).abs()
    assert bool((off <= bound + 1e-300).all()), f"off by {float((off - bound).max())} more than allowed, {float(off.max())} in all"


def _routing(ntokens, nexperts, topk, drop, seed):
    """(scatter_index, splits) through the library, and the pairs that have a row."""
    import flux_b200 as flux

    g = torch.Generator().manual_seed(seed)
    chosen = torch.rand(ntokens, nexperts, generator=g).topk(topk, dim=1).indices.to(torch.int32)
    if drop:
        chosen[torch.rand(ntokens, topk, generator=g) < drop] = -1
        chosen[torch.rand(ntokens, generator=g) < drop / 2] = -1
    si, splits = flux.calc_scatter_index(chosen.cuda(), torch.empty(nexperts), return_splits=True)
    return si, splits, chosen


# ---------------------------------------------------------------------------------------------------------------- route
def _route64(logits, topk):
    z = logits.double()
    order = torch.where(z.isnan(), torch.full_like(z, float("inf")), z)
    nan_first = torch.argsort(z.isnan().to(torch.int8), dim=1, descending=True, stable=True)
    by = torch.gather(order, 1, nan_first)
    # NaN first, then by value, ties by expert
    key = torch.where(torch.gather(z, 1, nan_first).isnan(), torch.full_like(by, float("inf")), by)
    at = torch.argsort(key, dim=1, descending=True, stable=True)
    chosen = torch.gather(nan_first, 1, at)[:, :topk]
    top = torch.gather(z, 1, chosen)
    alive = ~(top == -float("inf"))
    p = torch.where(alive, torch.exp(top - top[:, :1]), torch.zeros_like(top))
    w = torch.where(alive, p / p.sum(1, keepdim=True), torch.zeros_like(p))
    return torch.where(alive, chosen, torch.full_like(chosen, -1)).to(torch.int32), w


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("ntokens,nexperts,topk", [(1, 1, 1), (1, 8, 2), (5, 8, 8), (33, 31, 3), (64, 33, 32), (1000, 64, 6),
                                                    (257, 65, 4), (130, 300, 8), (9, 1024, 32)])
def test_route(dtype, ntokens, nexperts, topk):
    import flux_b200 as flux

    g = torch.Generator().manual_seed(ntokens + nexperts)
    z = (torch.randn(ntokens, nexperts, generator=g) * 3).to(dtype)
    dw = torch.randn(ntokens, topk, generator=g)
    want_c, want_w = _route64(z, topk)
    x = z.cuda().requires_grad_(True)
    chosen, w = flux.moe_route(x, topk)
    assert chosen.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(chosen.cpu(), want_c)
    # z - z_max is rounded once (|z - z_max| < 32: 32 u of the exponential), expf is within 2 ulp (4 u), the sum of k
    # terms k u (and their 36 u again), the quotient u
    rel = (2 * 36 + topk + 2) * U
    _within(w.detach(), want_w, rel * want_w)
    (dz,) = torch.autograd.grad(w, x, dw.cuda())
    s = (want_w * dw.double()).sum(1, keepdim=True)
    want = torch.zeros(ntokens, nexperts, dtype=torch.float64).scatter_(1, want_c.long(), want_w * (dw.double() - s))
    # w and the sum over k products are off by `rel` each, three more roundings, and the one to the logits' type
    scale = (dw.abs().double() + (want_w * dw.abs().double()).sum(1, keepdim=True)) * want_w
    bound = torch.zeros_like(want).scatter_(1, want_c.long(), (2 * rel + (topk + 3) * U) * scale)
    low = torch.finfo(dtype).smallest_normal * _half_step(dtype)
    _within(dz, want, bound + _half_step(dtype) * (want.abs() + bound) + low)


@pytest.mark.parametrize("dtype", FLOATS)
def test_route_masks_ties_and_values_that_are_no_numbers(dtype):
    import flux_b200 as flux

    inf, nan = float("inf"), float("nan")
    z = torch.tensor([
        [1.0, 1.0, 1.0, 1.0, 1.0],             # ties: the lower experts
        [-0.0, 0.0, -0.0, -1.0, 0.0],          # both zeros are one value
        [-inf, -inf, -inf, -inf, -inf],        # a mask that leaves nothing
        [-inf, 2.0, -inf, -inf, -inf],         # ... that leaves one
        [torch.finfo(torch.float32).min] * 5,  # the type's lowest value is a value
        [0.0, nan, 1.0, -inf, 2.0],            # NaN is the largest, and spreads
        [0.0, inf, 1.0, 5.0, 2.0],
        [1e-40, 2e-40, 0.0, -1e-40, -inf],     # subnormal differences count
    ]).to(dtype)
    if dtype != torch.float32:
        z[4] = torch.finfo(dtype).min
    chosen, w = flux.moe_route(z.cuda(), 3)
    want_c, want_w = _route64(z, 3)
    assert torch.equal(chosen.cpu(), want_c)
    assert torch.equal(w.cpu().isnan(), want_w.isnan())
    ok = ~want_w.isnan()
    _within(w.cpu()[ok], want_w[ok], 80 * U * want_w[ok])
    assert chosen[2].tolist() == [-1, -1, -1] and w[2].tolist() == [0.0, 0.0, 0.0]
    assert chosen[3].tolist() == [1, -1, -1] and w[3].tolist() == [1.0, 0.0, 0.0]
    # no gradient comes from what was not chosen
    x = z[:5].cuda().requires_grad_(True)
    _, w = flux.moe_route(x, 3)
    (dz,) = torch.autograd.grad(w, x, torch.full((5, 3), nan).where(chosen[:5].cpu() < 0, torch.ones(5, 3)).cuda())
    assert bool(dz.isfinite().all()) and float(dz[2:4].abs().max()) <= 4 * U


def test_route_gradient_against_differences():
    import flux_b200 as flux

    g = torch.Generator().manual_seed(3)
    z = torch.randn(6, 12, generator=g) * 2
    dw = torch.randn(6, 4, generator=g)
    x = z.cuda().requires_grad_(True)
    _, w = flux.moe_route(x, 4)
    (dz,) = torch.autograd.grad(w, x, dw.cuda())
    h = 1e-5
    for t, e in [(0, 3), (2, 0), (5, 11), (4, 7)]:
        up, down = z.double().clone(), z.double().clone()
        up[t, e] += h
        down[t, e] -= h
        diff = sum(sign * (_route64(v, 4)[1] * dw.double()).sum() for sign, v in ((1, up), (-1, down))) / (2 * h)
        # central differences of a softmax with |dw| < 4: h^2 / 6 times its third derivative (< 8 |dw| sums), fp32 results
        assert abs(float(diff) - float(dz[t, e])) < 1e-5


# ----------------------------------------------------------------------------------------------------- permute, unpermute
SIZES = [(1, 4, 1, 1), (1, 8, 2, 4096), (3, 8, 2, 2), (7, 16, 5, 33), (130, 8, 2, 64), (33, 64, 9, 130), (257, 32, 4, 1000), (20, 300, 12, 4100),
         (5000, 16, 3, 264), (6000, 8, 2, 36), (3001, 64, 10, 16)]


def _pairs(si):
    """(token, choice, row) of every pair that has a row."""
    si = si.cpu().long()
    t, j = (si >= 0).nonzero(as_tuple=True)
    return t, j, si[t, j]


@pytest.mark.parametrize("drop", [0.0, 0.3])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("ntokens,nexperts,topk,hidden", SIZES)
def test_permute_and_back_with_gradients(ntokens, nexperts, topk, hidden, dtype, drop):
    import flux_b200 as flux

    si, splits, _ = _routing(ntokens, nexperts, topk, drop, ntokens + hidden)
    t, j, r = _pairs(si)
    g = torch.Generator().manual_seed(hidden)
    rows = ntokens * topk
    x, y = torch.randn(ntokens, hidden, generator=g).to(dtype), torch.randn(rows, hidden, generator=g).to(dtype)
    drows, dout = torch.randn(rows, hidden, generator=g).to(dtype), torch.randn(ntokens, hidden, generator=g).to(dtype)
    wtype = {torch.float32: torch.float32, torch.bfloat16: torch.float32, torch.float16: torch.float16}[dtype]
    w = torch.rand(ntokens, topk, generator=g).to(wtype)
    # what belongs to nobody may hold anything
    n = int(splits.sum())
    assert n == r.numel()
    y[n:] = float("nan")
    drows[n:] = float("inf")
    wd = w.clone()
    wd[si.cpu() < 0] = float("nan")

    xg, yg, wg = (v.cuda().requires_grad_(True) for v in (x, y, wd))
    got = flux.moe_permute(xg, splits, si)
    want = torch.zeros(rows, hidden, dtype=dtype)
    want[r] = x[t]
    assert torch.equal(got.detach().cpu(), want)

    out = flux.moe_unpermute(yg, splits, si, wg)
    term = y[r].double() * w[t, j].double()[:, None]
    want = torch.zeros(ntokens, hidden, dtype=torch.float64).index_add_(0, t, term)
    size = torch.zeros_like(want).index_add_(0, t, term.abs())
    bound = 2 * topk * U * size
    half, low = _half_step(dtype), torch.finfo(dtype).smallest_normal * _half_step(dtype)
    _within(out.detach(), want, bound + half * (want.abs() + bound) + low)

    plain = flux.moe_unpermute(yg, splits, si)
    want = torch.zeros(ntokens, hidden, dtype=torch.float64).index_add_(0, t, y[r].double())
    size = torch.zeros_like(want).index_add_(0, t, y[r].double().abs())
    _within(plain.detach(), want, topk * U * size + half * (want.abs() + topk * U * size) + low)

    dx, dy, dw = torch.autograd.grad((got, out), (xg, yg, wg), (drows.cuda(), dout.cuda()))
    assert dx.dtype == dtype and dy.dtype == dtype and dw.dtype == wtype
    want = torch.zeros(ntokens, hidden, dtype=torch.float64).index_add_(0, t, drows[r].double())
    size = torch.zeros_like(want).index_add_(0, t, drows[r].double().abs())
    _within(dx, want, topk * U * size + half * (want.abs() + topk * U * size) + low)
    want = torch.zeros(rows, hidden, dtype=torch.float64)
    want[r] = dout[t].double() * w[t, j].double()[:, None]
    _within(dy, want, (U + half) * want.abs() * 1.001 + low)
    term = y[r].double() * dout[t].double()
    want, size = torch.zeros(ntokens, topk, dtype=torch.float64), torch.zeros(ntokens, topk, dtype=torch.float64)
    want[t, j], size[t, j] = term.sum(1), term.abs().sum(1)
    bound = (hidden + 1) * U * size
    _within(dw, want, bound + _half_step(wtype) * (want.abs() + bound))
    # only one of the two gradients
    y1 = y.cuda().requires_grad_(True)
    (dy1,) = torch.autograd.grad(flux.moe_unpermute(y1, splits, si, wd.cuda()), y1, dout.cuda())
    assert torch.equal(dy1, dy)
    (dw1,) = torch.autograd.grad(flux.moe_unpermute(y.cuda(), splits, si, wg), wg, dout.cuda())
    assert torch.equal(dw1, dw)
    (dy2,) = torch.autograd.grad(flux.moe_unpermute(y1, splits, si), y1, dout.cuda())
    want = torch.zeros(rows, hidden, dtype=dtype)
    want[r] = dout[t]
    assert torch.equal(dy2.cpu(), want)


def test_unpermute_gradients_against_differences():
    import flux_b200 as flux

    si, splits, _ = _routing(9, 8, 3, 0.2, 5)
    t, j, r = _pairs(si)
    g = torch.Generator().manual_seed(1)
    y, w, dout = torch.randn(27, 10, generator=g), torch.rand(9, 3, generator=g), torch.randn(9, 10, generator=g)
    yg, wg = y.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    dy, dw = torch.autograd.grad(flux.moe_unpermute(yg, splits, si, wg), (yg, wg), dout.cuda())

    def loss(y, w):
        out = torch.zeros(9, 10, dtype=torch.float64).index_add_(0, t, y[r].double() * w[t, j].double()[:, None])
        return float((out * dout.double()).sum())

    for p, grad, spots in ((0, dy, [(0, 0), (11, 9), (26, 4)]), (1, dw, [(0, 0), (4, 2), (8, 1)])):
        for at in spots:
            pair = [y.double().clone(), w.double().clone()]
            pair[p][at] += 0.5
            up = loss(*pair)
            pair[p][at] -= 1.0
            # linear in each: the difference is the gradient, but for 10 fp32 products of values below 5
            assert abs(up - loss(*pair) - float(grad[at])) < 10 * 25 * 4 * U


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int32, torch.int64, torch.float8_e4m3fn, torch.float64, torch.bool])
@pytest.mark.parametrize("hidden", [1, 3, 48, 1025])
def test_permute_moves_rows_of_any_type(dtype, hidden):
    import flux_b200 as flux

    si, splits, _ = _routing(40, 8, 2, 0.1, hidden)
    t, _, r = _pairs(si)
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 2 if dtype == torch.bool else 256, (40, hidden * size), generator=torch.Generator().manual_seed(2), dtype=torch.uint8)
    got = flux.moe_permute(raw.view(dtype).cuda(), splits, si)
    want = torch.zeros(80, hidden * size, dtype=torch.uint8)
    want[r] = raw[t]
    assert got.dtype == dtype and torch.equal(got.cpu().view(torch.uint8), want)


def test_layouts_and_alignments():
    """Strided, transposed and expanded inputs, and views that start between the vectors' boundaries."""
    import flux_b200 as flux

    si, splits, _ = _routing(24, 8, 2, 0.0, 9)
    g = torch.Generator().manual_seed(4)
    big = torch.randn(24, 200, generator=g).to(torch.bfloat16).cuda()
    t, j, r = _pairs(si)
    for x in (big[:, 3:67], big[:, ::2], big[:, :1].expand(24, 32), big.t().contiguous().t(), big.reshape(-1)[1:24 * 64 + 1].view(24, 64)):
        got = flux.moe_permute(x, splits, si).cpu()
        assert torch.equal(got[r], x.cpu()[t])
    y = torch.randn(48 * 64 + 1, generator=g).to(torch.float16).cuda()[1:].view(48, 64).requires_grad_(True)
    w = torch.rand(2, 24, generator=g).cuda().t().requires_grad_(True)
    dout = torch.randn(24, 1, generator=g).to(torch.float16).cuda().expand(24, 64)
    dy, dw = torch.autograd.grad(flux.moe_unpermute(y, splits, si, w), (y, w), dout)
    want = (dout.double().cpu()[t] * w.detach().double().cpu()[t, j][:, None])
    _within(dy.cpu()[r], want, (U + 2.0 ** -11) * 1.001 * want.abs() + 2.0 ** -25)
    term = y.detach().double().cpu()[r] * dout.double().cpu()[t]
    _within(dw.cpu()[t, j], term.sum(1), 65 * U * term.abs().sum(1))


def test_no_tokens():
    import flux_b200 as flux

    splits, si = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.empty((0, 2), dtype=torch.int32, device="cuda")
    x = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    rows = flux.moe_permute(x, splits, si)
    w = torch.empty((0, 2), device="cuda", requires_grad=True)
    out = flux.moe_unpermute(rows, splits, si, w)
    assert rows.shape == (0, 16) and out.shape == (0, 16)
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
    assert dx.shape == (0, 16) and dw.shape == (0, 2)
    chosen, weights = flux.moe_route(torch.empty((0, 8), device="cuda"), 2)
    assert chosen.shape == (0, 2) and weights.shape == (0, 2)


def test_pairs_without_an_expert_have_no_row():
    import flux_b200 as flux

    chosen = torch.tensor([[0, -1], [7, 2], [2, 4], [-3, 1 << 20]], dtype=torch.int32)
    si, splits = flux.calc_scatter_index(chosen.cuda(), torch.empty(4), return_splits=True)
    assert si.tolist() == [[0, -1], [-1, 1], [2, -1], [-1, -1]]
    assert splits.tolist() == [1, 0, 2, 0]


def test_training_chain_on_a_stream_and_in_a_graph():
    """Router to output and back, eager on a stream of its own, then captured and replayed with other inputs."""
    import flux_b200 as flux

    tokens, experts, topk, hidden = 96, 8, 2, 128
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(tokens, hidden, generator=g, device="cuda", requires_grad=True)
    router = torch.randn(experts, hidden, generator=g, device="cuda", requires_grad=True)
    dout = torch.randn(tokens, hidden, generator=g, device="cuda")
    counts = torch.empty(experts, dtype=torch.int32, device="cuda")

    def step():
        chosen, w = flux.moe_route(x @ router.t(), topk)
        si, splits = flux.calc_scatter_index(chosen, counts, return_splits=True)
        rows = flux.moe_permute(x, splits, si)
        out = flux.moe_unpermute(torch.tanh(rows), splits, si, w)
        return (out,) + torch.autograd.grad(out, (x, router), dout)

    def definition(x, router):
        x, router = x.detach().double().requires_grad_(True), router.detach().double().requires_grad_(True)
        top, chosen = torch.topk(x @ router.t(), topk, dim=1)
        out = torch.tanh(x) * torch.softmax(top, 1).sum(1, keepdim=True)
        return (out,) + torch.autograd.grad(out, (x, router), dout.double())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for a, b in zip([v.detach() for v in got], [v.detach() for v in definition(x, router)]):
        # sums of at most hidden or tokens products and a few elementwise steps in fp32
        assert float((a - b).abs().max()) <= 4 * hidden * U * float(b.abs().max() + 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    with torch.no_grad():
        x.copy_(torch.randn(tokens, hidden, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip([v.detach() for v in captured], [v.detach() for v in definition(x, router)]):
        assert float((a - b).abs().max()) <= 4 * hidden * U * float(b.abs().max() + 1)


def test_results_do_not_change_from_run_to_run():
    import flux_b200 as flux

    si, splits, _ = _routing(500, 16, 4, 0.1, 8)
    g = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randn(2000, 520, generator=g, device="cuda", requires_grad=True)
    w = torch.rand(500, 4, generator=g, device="cuda", requires_grad=True)
    dout = torch.randn(500, 520, generator=g, device="cuda")
    runs = []
    for _ in range(3):
        out = flux.moe_unpermute(y, splits, si, w)
        runs.append((out,) + torch.autograd.grad(out, (y, w), dout))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("hidden", [4096, 4100, 4097])
def test_more_than_31_bits_of_values(hidden):
    import flux_b200 as flux

    ntokens, topk, dtype = 66000, 8, torch.bfloat16
    si, splits, _ = _routing(ntokens, 16, topk, 0.01, hidden)
    last = int(splits.sum())
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x = torch.randn(ntokens, hidden, generator=g, device="cuda", dtype=dtype)
    dout = torch.randn(ntokens, hidden, generator=g, device="cuda", dtype=dtype)
    w = torch.rand(ntokens, topk, generator=g, device="cuda").requires_grad_(True)
    rows = flux.moe_permute(x, splits, si).requires_grad_(True)
    out = flux.moe_unpermute(rows, splits, si, w)
    drows, dw = torch.autograd.grad(out, (rows, w), dout)
    (dx,) = torch.autograd.grad(flux.moe_permute(x.requires_grad_(True), splits, si), x, drows)
    assert int(rows[last:].count_nonzero()) == 0 and int(drows[last:].count_nonzero()) == 0
    half, low = _half_step(dtype), torch.finfo(dtype).smallest_normal
    for at in (slice(0, 100), slice(ntokens // 2, ntokens // 2 + 100), slice(ntokens - 100, ntokens)):
        t, j, r = _pairs(si[at])
        xs, gs, ws = x[at].detach().cpu(), dout[at].cpu().double(), w[at].detach().cpu().double()
        here = r.cuda()
        assert torch.equal(rows[here].cpu(), xs[t])
        total = torch.zeros(100, dtype=torch.float64).index_add_(0, t, ws[t, j])[:, None]
        want = xs.double() * total
        _within(out[at].detach(), want, 2 * topk * U * want.abs() + half * want.abs() * 1.001 + low)
        want = gs[t] * ws[t, j][:, None]
        _within(drows[here], want, (U + half) * want.abs() * 1.001 + low)
        term = xs[t].double() * gs[t]
        want, size = torch.zeros(100, topk, dtype=torch.float64), torch.zeros(100, topk, dtype=torch.float64)
        want[t, j], size[t, j] = term.sum(1), term.abs().sum(1)
        _within(dw[at], want, (hidden + 2) * U * size)
        term = drows[here].cpu().double()
        want = torch.zeros(100, hidden, dtype=torch.float64).index_add_(0, t, term)
        size = torch.zeros(100, hidden, dtype=torch.float64).index_add_(0, t, term.abs())
        _within(dx[at], want, topk * U * size + half * (want.abs() + topk * U * size) + low)


def test_gradients_and_tokens_as_torch_hands_them_over():
    """Expanded and transposed gradients, and tokens whose conjugation is only marked."""
    import flux_b200 as flux

    si, splits, _ = _routing(37, 8, 2, 0.2, 11)
    z = torch.randn(37, 8, device="cuda", requires_grad=True)
    _, w = flux.moe_route(z, 2)
    dw = torch.randn(2, 37, device="cuda")
    (dense,) = torch.autograd.grad(w, z, dw.t().contiguous(), retain_graph=True)
    (strided,) = torch.autograd.grad(w, z, dw.t(), retain_graph=True)
    (ones,) = torch.autograd.grad(w, z, torch.ones_like(w), retain_graph=True)
    (expanded,) = torch.autograd.grad(w.sum(), z)
    assert torch.equal(dense, strided) and torch.equal(ones, expanded)
    x = torch.randn(37, 5, device="cuda", dtype=torch.complex64)
    for t in (x.conj(), x.conj().t().contiguous().t(), x.conj().imag, x[:, :1].conj().imag):
        assert torch.equal(flux.moe_permute(t, splits, si), flux.moe_permute(t.resolve_conj().resolve_neg().contiguous(), splits, si))
    one = torch.randn(1, 1, device="cuda", dtype=torch.complex64).conj().imag
    index, counts = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    assert one.is_neg() and torch.equal(flux.moe_permute(one, counts, index), one) and torch.equal(flux.moe_unpermute(one, counts, index), one)
