"""The layers with microscaled 4-bit weights: what a layer returns is what its operators return one after the other, bit for
bit, and every operator of the run is what its definition makes of the operator before it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _close(got, want, size, terms, dtype):
    """`terms` products summed in fp32 by adders that round or cut, and one rounding to `dtype`."""
    off = terms * 2.0 ** -23 * size
    off = off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got.double() - want).abs() <= off).all())


def _experts(rows, weights, splits):
    out, size, r = [], [], 0
    for e, n in enumerate(splits.tolist()):
        out.append(rows[r:r + n] @ weights[e].t())
        size.append(rows[r:r + n].abs() @ weights[e].abs().t())
        r += n
    return torch.cat(out), torch.cat(size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden,ffn,experts,topk,gated", [(1, 256, 128, 8, 2, True), (40, 512, 320, 8, 2, False), (300, 256, 416, 16, 4, True),
                                                                  (7, 96, 64, 4, 4, False)])
def test_moe_layer(tokens, hidden, ffn, experts, topk, gated, dtype):
    import flux_b200 as flux

    torch.manual_seed(tokens)
    moe = flux.MoEMLP(hidden, ffn, experts, topk, tokens, None, gated=gated, dtype=dtype)
    layer = flux.MXMoEMLP.from_moe(moe)
    x = torch.randn(tokens, hidden, device="cuda", dtype=dtype)
    got = layer(x)
    assert got.shape == x.shape and got.dtype == dtype

    with torch.no_grad():
        logits = x.float() @ moe.router.t()
        chosen, weights = flux.moe_route(logits, topk)
        top, idx = torch.topk(logits, topk, dim=1)
        assert torch.equal(chosen.long(), idx)
        assert float((weights.double() - torch.softmax(top.double(), 1)).abs().max()) < 100 * 2.0 ** -24
        si, splits = flux.calc_scatter_index(chosen, torch.empty(experts), return_splits=True)
        up = flux.mx_quantize(torch.cat((moe.w_gate, moe.w_up), 1) if gated else moe.w_up)
        down = flux.mx_quantize(moe.w_down)
        rows = flux.mx_quantize(x, splits, si)
        source = torch.argsort(si.view(-1)) // topk
        assert torch.equal(rows.dequantize(torch.float32), flux.mx_quantize(x).dequantize(torch.float32)[source])
        h = flux.mx_grouped_gemm(rows, up, splits, dtype)
        want, size = _experts(rows.dequantize(torch.float32).double(), up.dequantize(torch.float32).double(), splits)
        _close(h, want, size, hidden, dtype)
        act = torch.nn.functional.silu(h[:, :ffn]) * h[:, ffn:] if gated else torch.nn.functional.gelu(h)
        q = flux.mx_quantize(act)
        y = flux.mx_grouped_gemm(q, down, splits, dtype)
        want, size = _experts(q.dequantize(torch.float32).double(), down.dequantize(torch.float32).double(), splits)
        _close(y, want, size, ffn, dtype)
        out = flux.moe_unpermute(y, splits, si, weights)
        term = y.double()[si.long()] * weights.double()[..., None]
        _close(out, term.sum(1), term.abs().sum(1), 2 * topk, dtype)
    torch.cuda.synchronize()
    flux.get_comm(None).check_status()
    assert torch.equal(out, got)
    # three dimensions, and the same from a state dict
    assert torch.equal(layer(x.view(1, tokens, hidden))[0], got)
    other = flux.MXMoEMLP.from_moe(flux.MoEMLP(hidden, ffn, experts, topk, tokens, None, gated=gated, dtype=dtype))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), got)


@pytest.mark.parametrize("bias", [False, True])
def test_linear(bias):
    import flux_b200 as flux

    torch.manual_seed(1)
    linear = torch.nn.Linear(256, 200, bias=bias, device="cuda", dtype=torch.bfloat16)
    layer = flux.MXLinear.from_linear(linear)
    x = torch.randn(3, 5, 256, device="cuda", dtype=torch.bfloat16)
    y = layer(x)
    xv, wv = (flux.mx_quantize(v.detach()).dequantize(torch.float32).double() for v in (x, linear.weight))
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias:
        want, size = want + linear.bias.double(), size + linear.bias.double().abs()
    assert y.shape == (3, 5, 200) and not y.requires_grad
    _close(y.detach(), want.detach(), size.detach(), 257, torch.bfloat16)
    assert layer.weight_data.numel() * 2 == linear.weight.numel()
    # quantised elsewhere
    q = flux.mx_quantize(linear.weight.detach())
    again = flux.MXLinear(flux.MXTensor(q.data, q.scales), linear.bias, output_dtype=torch.bfloat16)
    assert torch.equal(again(x), y)


def test_moe_layer_captured_and_replayed():
    import flux_b200 as flux

    torch.manual_seed(2)
    layer = flux.MXMoEMLP.from_moe(flux.MoEMLP(256, 512, 8, 2, 64, None, gated=True, dtype=torch.bfloat16))
    x = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(x)
    for seed in range(3):
        x.copy_(torch.randn(64, 256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x))
    flux.get_comm(None).check_status()


def test_no_tokens():
    import flux_b200 as flux

    layer = flux.MXMoEMLP.from_moe(flux.MoEMLP(128, 64, 4, 2, 8, None, dtype=torch.bfloat16))
    x = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16)
    assert layer(x).shape == (0, 128)
    assert flux.MXLinear(torch.randn(48, 128, device="cuda"))(x).shape == (0, 48)
    torch.cuda.synchronize()


def test_layers_refuse_what_does_not_fit():
    import flux_b200 as flux

    moe = flux.MoEMLP(256, 512, 8, 2, 64, None, dtype=torch.bfloat16)
    moe.world = 2
    with pytest.raises(RuntimeError, match="several ranks"):
        flux.MXMoEMLP.from_moe(moe)
    column = flux.ColumnParallelLinear(256, 512, 64, None)
    column.world = 2
    with pytest.raises(RuntimeError, match="several ranks"):
        flux.MXLinear.from_linear(column)
    with pytest.raises(RuntimeError, match="do not fit together"):
        flux.MXMoEMLP(moe.router, moe.w_up, moe.w_up, 2)
    with pytest.raises(RuntimeError, match="must be"):
        flux.MXLinear(moe.w_up)


def test_the_path_from_several_threads():
    """Each thread with a stream and sizes of its own; what it gets the first time, alone or not, it gets every time."""
    import threading

    import flux_b200 as flux

    flux.init_flux_shm(None)
    wrong = []

    def work(i):
        try:
            g = torch.Generator(device="cuda")
            with torch.cuda.stream(torch.cuda.Stream()):
                first = None
                for _ in range(12):
                    g.manual_seed(i)
                    tokens, hidden = 50 + 37 * i, 512 + 32 * i
                    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16().requires_grad_(True)
                    chosen, weights = flux.moe_route(torch.randn(tokens, 8, device="cuda", generator=g), 2)
                    si, splits = flux.calc_scatter_index(chosen, torch.empty(8), return_splits=True)
                    rows = flux.moe_permute(x, splits, si)
                    out = flux.moe_unpermute(rows, splits, si, weights)
                    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
                    up = flux.mx_quantize(torch.randn(8, 300 + i, hidden, device="cuda", generator=g))
                    w = flux.mx_quantize(torch.randn(700 + i, hidden, device="cuda", generator=g))
                    got = [chosen, weights, rows.detach(), out.detach(), dx, flux.mx_grouped_gemm(flux.mx_quantize(x.detach(), splits, si), up, splits),
                           flux.mx_gemm(flux.mx_quantize(x.detach()), w)]
                    first = first or got
                    wrong.extend((i, n) for n, (a, b) in enumerate(zip(first, got)) if not torch.equal(a, b))
        except Exception as e:  # (an exception in a thread is not pytest's)
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    flux.get_comm(None).check_status()
    assert wrong == []


FIRST_PRODUCTS = """
import threading, torch, flux_b200 as flux
from flux_b200 import mx
q = [flux.mx_quantize(torch.randn(40 + i, 256, device="cuda")) for i in range(6)]
w, splits = flux.mx_quantize(torch.randn(2, 96, 256, device="cuda")), torch.tensor([30, 10], dtype=torch.int32, device="cuda")
one = flux.MXTensor(w.data[0], w.scales[0])
torch.cuda.synchronize()
start, got = threading.Barrier(6), [None] * 6
def work(i):
    torch.cuda.set_device(0)
    start.wait()
    got[i] = flux.mx_gemm(q[i], one) if i % 2 else flux.mx_grouped_gemm(q[i], w, splits)
threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
flux.mx_check_status()
for i in range(6):
    again = flux.mx_gemm(q[i], one) if i % 2 else flux.mx_grouped_gemm(q[i], w, splits)
    rows = 40 + i if i % 2 else 40
    assert torch.equal(got[i][:rows], again[:rows])
print("same")
"""


def test_first_products_of_several_threads():
    """Of a process without a communicator: the threads make one together."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_PRODUCTS], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr[-2000:]
