"""Refusals of the microscaled operators: they need no GPU."""
import ctypes as C

import pytest
import torch

import flux_b200 as flux
from flux_b200 import _lib


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError, match="mx_quantize: x must be"):
        flux.mx_quantize(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="MXTensor: data and scales"):
        flux.MXTensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="mx_gemm: operands"):
        flux.mx_gemm(torch.zeros(4, 64), torch.zeros(8, 64))
    with pytest.raises(RuntimeError, match="mx_grouped_gemm: operands"):
        flux.mx_grouped_gemm(torch.zeros(4, 64), torch.zeros(2, 8, 64), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="mx_dequantize: q"):
        flux.mx_dequantize(torch.zeros(4, 64))


P = C.c_void_p(256)  # never read: the calls are refused first


@pytest.mark.parametrize("change,words", [
    ({"dtype": _lib.E4M3}, "fp32, bf16 or fp16"), ({"rows": -1}, "rows=-1"), ({"batch": -1}, "batch=-1"), ({"k": 0}, "k=0"), ({"k": 48}, "k=48"),
    ({"batch": 1 << 16, "rows": 1 << 15}, "too many"), ({"splits": P}, "belong together"), ({"index": P}, "belong together"),
    ({"splits": P, "index": P, "topk": 0}, "topk=0"), ({"splits": P, "index": P, "batch": 2}, "batch=2"), ({"splits": P, "index": P, "nexperts": 0}, "nexperts=0"),
    ({"splits": P, "index": P, "rows": 1 << 29}, "too many"), ({"x": None}, "NULL"), ({"data": None}, "NULL"), ({"scales": None}, "NULL"),
    ({"x": C.c_void_p(257)}, "aligned"), ({"data": C.c_void_p(260)}, "aligned"), ({"scales": C.c_void_p(258)}, "aligned"),
])
def test_quantize_arguments(change, words):
    a = {"x": P, "dtype": _lib.BF16, "batch": 1, "rows": 4, "k": 64, "ldx": 64, "data": P, "scales": P, "splits": None, "nexperts": 8, "index": None,
         "topk": 2, **change}
    assert _lib.load().fluxb_mx_quantize(a["x"], a["dtype"], a["batch"], a["rows"], a["k"], a["ldx"], a["data"], a["scales"], a["splits"], a["nexperts"],
                                         a["index"], a["topk"], None) == _lib.FLUXB_ERR_INVALID
    assert "mx_quantize" in _lib.last_error() and words in _lib.last_error()


@pytest.mark.parametrize("change,words", [({"dtype": _lib.S8}, "fp32, bf16 or fp16"), ({"rows": -1}, "rows=-1"), ({"k": 33}, "k=33"),
                                          ({"data": None}, "NULL"), ({"data": C.c_void_p(258)}, "aligned"), ({"out": C.c_void_p(264)}, "aligned")])
def test_dequantize_arguments(change, words):
    a = {"data": P, "scales": P, "rows": 4, "k": 64, "dtype": _lib.BF16, "out": P, **change}
    assert _lib.load().fluxb_mx_dequantize(a["data"], a["scales"], 1, a["rows"], a["k"], a["dtype"], a["out"], None) == _lib.FLUXB_ERR_INVALID
    assert "mx_dequantize" in _lib.last_error() and words in _lib.last_error()


@pytest.mark.parametrize("change,words", [
    ({"comm": None}, "NULL"), ({"xq": None}, "NULL"), ({"out": None}, "NULL"), ({"k": 16}, "k=16"), ({"k": 80}, "k=80"), ({"n": 0}, "n=0"), ({"m": -1}, "=-1"),
    ({"xq": C.c_void_p(264)}, "16-byte"), ({"ws": C.c_void_p(264)}, "16-byte"), ({"dtype": _lib.E5M2}, "not bf16/f16/f32"),
    ({"out": C.c_void_p(257)}, "aligned to its type"), ({"dtype": _lib.F32, "out": C.c_void_p(258)}, "aligned to its type"),
])
def test_product_arguments(change, words):
    a = {"comm": P, "xq": P, "xs": P, "wq": P, "ws": P, "out": P, "m": 4, "n": 8, "k": 64, "dtype": _lib.BF16, **change}
    lib = _lib.load()
    assert lib.fluxb_mx_gemm(a["comm"], a["xq"], a["xs"], a["wq"], a["ws"], a["out"], a["m"], a["n"], a["k"], a["dtype"], None, None, None) == _lib.FLUXB_ERR_INVALID
    assert words in _lib.last_error()
    assert lib.fluxb_mx_grouped_gemm(a["comm"], a["xq"], a["xs"], a["m"], a["wq"], a["ws"], 4, P, a["out"], a["n"], a["k"], a["dtype"], P, None,
                                     None) == _lib.FLUXB_ERR_INVALID
    assert words in _lib.last_error()


@pytest.mark.parametrize("change", [{"m": (1 << 31) - 1}, {"m": (1 << 31) - 512}, {"n": (1 << 31) - 1}])
def test_rows_whose_tiles_would_pass_31_bits(change):
    a = {"m": 4, "n": 8, **change}
    lib = _lib.load()
    assert lib.fluxb_mx_gemm(P, P, P, P, P, P, a["m"], a["n"], 32, _lib.BF16, None, None, None) == _lib.FLUXB_ERR_INVALID
    assert "invalid" in _lib.last_error()
    assert lib.fluxb_mx_grouped_gemm(P, P, P, a["m"], P, P, 1, P, P, a["n"], 32, _lib.BF16, P, None, None) == _lib.FLUXB_ERR_INVALID
    assert "invalid" in _lib.last_error() or "too many" in _lib.last_error()


def test_grouped_arguments():
    lib = _lib.load()
    for nexperts, n, splits, ws, words in ((0, 8, P, P, "nexperts=0"), (1025, 8, P, P, "nexperts=1025"), (4, 8, None, P, "NULL"), (4, 8, P, None, "NULL"),
                                           (4, 8, P, C.c_void_p(264), "workspace"), (1024, 1 << 22, P, P, "too many")):
        assert lib.fluxb_mx_grouped_gemm(P, P, P, 4, P, P, nexperts, splits, P, n, 64, _lib.BF16, ws, None, None) == _lib.FLUXB_ERR_INVALID
        assert words in _lib.last_error()


def test_sizes():
    lib = _lib.load()
    assert lib.fluxb_mx_scale_bytes(1, 1, 32) == 512 and lib.fluxb_mx_scale_bytes(3, 129, 160) == 3 * 2 * 2 * 512 and lib.fluxb_mx_scale_bytes(1, 0, 64) == 0
    # for every tile width: the rows' whole tiles and one begun for each expert that can have rows, one or two blocks each
    for rows, nexperts in ((300, 5), (4, 1024), (100000, 64), (1, 1)):
        most = max((rows // bn + min(nexperts, rows)) * -(-bn // 128) for bn in (64, 128, 192, 256))
        assert lib.fluxb_mx_grouped_workspace_bytes(rows, nexperts, 160) >= most * 2 * 512
    assert lib.fluxb_mx_scale_bytes(-1, 4, 64) == 0 and lib.fluxb_mx_grouped_workspace_bytes(4, -1, 64) == 0


def _far(*shape, dtype=torch.uint8):
    """A tensor of any size without memory."""
    return torch.empty(shape, dtype=dtype, device="meta")


def test_sizes_that_do_not_fit_the_native_call(monkeypatch):
    """The library takes 32-bit sizes, and what passes them would arrive as another size: 2^32 + 32 as 32."""
    from flux_b200 import mx

    monkeypatch.setattr(mx, "_on_device", lambda t: True)
    monkeypatch.setattr(mx, "_cur_stream", lambda: None)
    for k in (1 << 31, (1 << 32) + 32):
        with pytest.raises(RuntimeError, match=f"K {k} is too large"):
            flux.mx_quantize(_far(1, k, dtype=torch.bfloat16))
        with pytest.raises(RuntimeError, match=f"K {k} is too large"):
            flux.MXTensor(_far(1, k // 2), _far(1, k // 32))
    for shape in ((1 << 31, 16), (1 << 16, 1 << 15, 16), ((1 << 32) + 4, 1, 16)):
        with pytest.raises(RuntimeError, match="rows are too many"):
            flux.MXTensor(_far(*shape), _far(*shape[:-1], 1))


def _stored(lead=(), rows=3, k=64):
    """An MXTensor as `mx_quantize` makes it, values and scales in one allocation, in host memory."""
    from flux_b200 import mx

    t = mx.MXTensor.__new__(mx.MXTensor)
    t.lead, t.rows, t.k, t._dev = lead, rows, k, -1
    n = rows * k // 2
    for d in lead:
        n *= d
    at = (n + 15) & ~15
    blocks = mx._blocks_shape(lead, rows, k)
    t._store = torch.randint(0, 256, (at + torch.Size(blocks).numel(),), dtype=torch.uint8)
    t._data = t._blocks = None
    t._data_ptr = t._store.data_ptr()
    t._blocks_ptr = t._data_ptr + at
    return t


@pytest.mark.parametrize("how", ["deepcopy", "copy", "pickle", "torch.save"])
@pytest.mark.parametrize("lead", [(), (2, 3)])
def test_copies_point_to_their_own_memory(how, lead):
    """A copy's addresses are those of the copy's tensors, not those of tensors that may be gone by the time it is used."""
    import copy
    import io
    import pickle

    q = _stored(lead)
    if how == "torch.save":
        f = io.BytesIO()
        torch.save(q, f)
        f.seek(0)
        c = torch.load(f, weights_only=False)
    else:
        c = {"deepcopy": copy.deepcopy, "copy": copy.copy, "pickle": lambda t: pickle.loads(pickle.dumps(t))}[how](q)
    assert c.shape == q.shape and torch.equal(c.data, q.data) and torch.equal(c.blocks, q.blocks) and c._dev == q._dev
    assert (c._data_ptr, c._blocks_ptr) == (c.data.data_ptr(), c.blocks.data_ptr())
    assert (c._data_ptr == q._data_ptr) == (how == "copy")
    assert torch.equal(c.scales, q.scales)


def test_tokens_of_another_size_than_the_layer_are_refused():
    """Twice the layer's size used to be taken as twice as many tokens."""
    from flux_b200 import mx

    def weight(n, k):
        return mx.MXTensor._of(torch.zeros(2, n, k // 2, dtype=torch.uint8), torch.zeros(2, 1, 1, 512, dtype=torch.uint8))

    layer = flux.MXMoEMLP(torch.zeros(2, 64), weight(96, 64), weight(64, 96), 1)
    for shape in ((4, 128), (4, 32), (2, 3, 192), (0, 128), ()):
        with pytest.raises(RuntimeError, match=r"MXMoEMLP: .*\[\.\.\., 64\]"):
            layer(torch.zeros(shape))


def test_gate_and_up_projection_of_different_sizes_are_refused():
    """Both together have twice the experts' size, and would be cut in the middle."""
    with pytest.raises(RuntimeError, match="MXMoEMLP: w_gate"):
        flux.MXMoEMLP(torch.zeros(2, 64), torch.zeros(2, 128, 64), torch.zeros(2, 64, 96), 1, w_gate=torch.zeros(2, 64, 64))
    q = _stored((2,), 96, 64)
    with pytest.raises(RuntimeError, match="MXMoEMLP: w_gate"):
        flux.MXMoEMLP(torch.zeros(2, 64), q, q, 1, w_gate=q)
