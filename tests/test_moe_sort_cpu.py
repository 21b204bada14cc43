"""Refusals of the routing and sort operators: they need no GPU."""
import ctypes as C
import weakref

import pytest
import torch

import flux_b200 as flux
from flux_b200 import _lib


def test_tensors_off_the_gpu_are_refused():
    x, si, splits = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="moe_route: logits"):
        flux.moe_route(x, 2)
    with pytest.raises(RuntimeError, match="moe_permute: tokens"):
        flux.moe_permute(x, splits, si)
    with pytest.raises(RuntimeError, match="moe_unpermute: rows"):
        flux.moe_unpermute(torch.zeros(8, 8), splits, si)


@pytest.mark.parametrize("dtype,ntokens,nexperts,topk", [(_lib.E4M3, 4, 8, 2), (_lib.S8, 4, 8, 2), (_lib.F32, -1, 8, 2), (_lib.F32, 4, 0, 1),
                                                         (_lib.F32, 4, 1025, 2), (_lib.F32, 4, 8, 0), (_lib.F32, 4, 8, 9), (_lib.F32, 4, 64, 33),
                                                         (_lib.F32, 1 << 30, 8, 2), (_lib.F32, 4, 8, 2)])
def test_route_arguments(dtype, ntokens, nexperts, topk):
    lib = _lib.load()  # (the last case has NULL pointers only)
    assert lib.fluxb_moe_route(None, dtype, ntokens, nexperts, topk, None, None, None) == _lib.FLUXB_ERR_INVALID
    assert "moe_route" in _lib.last_error()
    assert lib.fluxb_moe_route_backward(None, None, None, dtype, ntokens, nexperts, topk, None, None) == _lib.FLUXB_ERR_INVALID
    assert "moe_route_backward" in _lib.last_error()


@pytest.mark.parametrize("ntokens,topk,size,nexperts", [(-1, 2, 64, 8), (4, 0, 64, 8), (4, 2, 0, 8), (1 << 29, 2, 64, 8), (4, 2, 1 << 30, 8),
                                                        (4, 2, 64, 0), (4, 2, 64, 8)])
def test_sort_arguments(ntokens, topk, size, nexperts):
    lib = _lib.load()
    assert lib.fluxb_moe_permute(None, ntokens, topk, size, None, nexperts, None, None, None) == _lib.FLUXB_ERR_INVALID
    assert "moe_permute" in _lib.last_error()
    if nexperts:
        assert lib.fluxb_moe_unpermute(None, _lib.BF16, ntokens, topk, size, None, None, 0, None, None) == _lib.FLUXB_ERR_INVALID
        assert "moe_unpermute" in _lib.last_error()
    assert lib.fluxb_moe_unpermute_backward(None, None, _lib.BF16, ntokens, topk, size, None, nexperts, None, None, _lib.F32, None, None,
                                            None) == _lib.FLUXB_ERR_INVALID
    assert "moe_unpermute_backward" in _lib.last_error()


def test_sort_types_and_null_pairs():
    lib = _lib.load()
    p = C.c_void_p(256)  # never read: the call is refused first
    assert lib.fluxb_moe_unpermute(p, _lib.E4M3, 4, 2, 64, p, None, 0, p, None) == _lib.FLUXB_ERR_INVALID
    assert lib.fluxb_moe_unpermute(p, _lib.BF16, 4, 2, 64, p, p, _lib.S8, p, None) == _lib.FLUXB_ERR_INVALID
    # the rows without the weights' gradient, and the other way round
    for rows, dw in ((p, None), (None, p)):
        assert lib.fluxb_moe_unpermute_backward(p, rows, _lib.BF16, 4, 2, 64, p, 8, p, p, _lib.F32, p, dw, None) == _lib.FLUXB_ERR_INVALID
        assert "gradient" in _lib.last_error()


def test_no_tokens_is_no_work():
    lib = _lib.load()
    assert lib.fluxb_moe_route(None, _lib.F32, 0, 8, 2, None, None, None) == _lib.FLUXB_OK
    assert lib.fluxb_moe_permute(None, 0, 2, 64, None, 8, None, None, None) == _lib.FLUXB_OK
    assert lib.fluxb_moe_unpermute(None, _lib.F32, 0, 2, 64, None, None, 0, None, None) == _lib.FLUXB_OK


class _Context:
    """What an autograd function sees of its forward pass."""

    def __init__(self, saved, **kept):
        self.saved_tensors = saved
        self.__dict__.update(kept)


def test_a_gradient_that_is_copied_lives_until_the_native_call_returns(monkeypatch):
    """An expanded gradient (as from `w.sum()`) is made contiguous: that copy is the kernel's input, and its memory must not go
    back to the allocator before the launch is queued."""
    from flux_b200 import moe

    copies, alive = [], []
    contiguous = torch.Tensor.contiguous

    def watched(t, *args, **kwargs):
        c = contiguous(t, *args, **kwargs)
        copies.append((c.data_ptr(), weakref.ref(c)))
        return c

    class Library:
        def fluxb_moe_route_backward(self, dweights, *_):
            alive.extend(ref() is not None for ptr, ref in copies if ptr == dweights)
            return _lib.FLUXB_OK

    monkeypatch.setattr(torch.Tensor, "contiguous", watched)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(moe, "_cur_stream", lambda: None)
    ctx = _Context((torch.zeros(3, 2, dtype=torch.int32), torch.full((3, 2), 0.5)), like=(torch.float32, 8))
    dlogits, _ = moe._RouteFn.backward(ctx, None, torch.ones(()).expand(3, 2))
    assert dlogits.shape == (3, 8) and alive == [True]


@pytest.mark.parametrize("counts_on_device", [False, True])
def test_indexes_that_are_copied_live_until_the_native_call_returns(monkeypatch, counts_on_device):
    from flux_b200 import moe

    copies, alive = [], []
    contiguous = torch.Tensor.contiguous

    def watched(t, *args, **kwargs):
        c = contiguous(t, *args, **kwargs)
        copies.append((c.data_ptr(), weakref.ref(c)))
        return c

    def launched(*args):
        alive.extend(ref() is not None for ptr, ref in copies if ptr in args)
        return _lib.FLUXB_OK

    class Library:
        fluxb_moe_gather_rs_forward_dev = fluxb_moe_gather_rs_forward_ep = staticmethod(launched)

    monkeypatch.setattr(torch.Tensor, "contiguous", watched)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(moe, "_check", lambda ok, what: None)  # (the tensors are not on a GPU)
    monkeypatch.setattr(moe, "_cur_stream", lambda: None)
    op = object.__new__(moe.GemmGroupedV3GatherRS)
    op.__dict__.update(comm=type("", (), {"world": 1}), ep_size=1, nexperts=2, n_dim=4, topk=2, max_m=6, input_dtype=torch.float32,
                       output_dtype=torch.float32, _h=None)
    index = torch.zeros(6, 2, dtype=torch.int32)[:, 0]
    counts = torch.zeros(2, 2, dtype=torch.int32)[:, 0]
    op._forward(torch.zeros(6, 8), torch.zeros(2, 4, 8), None if counts_on_device else counts, counts if counts_on_device else None, index)
    assert alive == [True, True]


def test_sizes_that_do_not_fit_the_native_call(monkeypatch):
    """The library takes 32-bit sizes, and what passes them would arrive as another size: 2^32 + 8 as 8."""
    from flux_b200 import moe

    monkeypatch.setattr(moe, "_on_device", lambda t: True)
    monkeypatch.setattr(moe, "_cur_stream", lambda: None)

    class Library:  # takes every call
        def __getattr__(self, name):
            return lambda *_: _lib.FLUXB_OK

    monkeypatch.setattr(_lib, "load", Library)

    def far(*shape, dtype=torch.float32):  # of any size, without memory
        return torch.empty(shape, dtype=dtype, device="meta")

    index, splits = far(4, 2, dtype=torch.int32), far(8, dtype=torch.int32)
    for experts in (1025, 1 << 31, (1 << 32) + 8):
        with pytest.raises(RuntimeError, match=f"moe_route: .*{experts} experts"):
            flux.moe_route(far(4, experts), 2)
    with pytest.raises(RuntimeError, match="moe_route: topk=33"):
        flux.moe_route(far(4, 64), 33)
    for hidden in (1 << 28, (1 << 32) + 64):
        with pytest.raises(RuntimeError, match=f"moe_unpermute: hidden={hidden}"):
            flux.moe_unpermute(far(8, hidden), splits, index)
    for experts in (1 << 31, (1 << 32) + 8):
        with pytest.raises(RuntimeError, match=f"{experts} experts"):
            flux.moe_permute(far(4, 8), far(experts, dtype=torch.int32), index)
    for topk in (1 << 30, (1 << 32) + 2):
        with pytest.raises(RuntimeError, match="too many"):
            flux.moe_permute(far(0, 8), splits, far(0, topk, dtype=torch.int32))
    flux.moe_route(far(4, 1024), 32), flux.moe_unpermute(far(8, (1 << 28) - 1), splits, index), flux.moe_permute(far(4, 8), splits, index)


def test_conjugations_and_signs_that_torch_has_put_off(monkeypatch):
    """`conj()` and what follows from it are marks on a tensor, which its memory does not show: the kernels get memory that holds
    the values."""
    from flux_b200 import moe

    seen = {}

    class Library:  # keeps what the first argument points to, of the size of the tensor under test
        def __getattr__(self, name):
            def call(first, *_):
                seen[name] = C.string_at(first, nbytes)
                return _lib.FLUXB_OK

            return call

    monkeypatch.setattr(_lib, "load", Library)
    for name in ("_on_device", "_cur_stream"):
        monkeypatch.setattr(moe, name, lambda *_: True)
    index, splits = torch.zeros(1, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)

    def bits(t):
        return t.resolve_conj().resolve_neg().clone(memory_format=torch.contiguous_format).numpy().tobytes()

    z = torch.randn(1, 5, dtype=torch.complex64)
    lazy = z.conj()
    assert lazy.is_conj() and lazy.is_contiguous()
    nbytes = 40
    flux.moe_permute(lazy, splits, index)
    assert seen["fluxb_moe_permute"] == bits(lazy) != bits(z)
    lazy = torch.randn(1, 1, dtype=torch.complex64).conj().imag
    assert lazy.is_neg() and lazy.is_contiguous()
    nbytes = 4
    flux.moe_permute(lazy, splits, index)
    flux.moe_unpermute(lazy, splits, index)
    flux.moe_route(lazy, 1)
    for name in ("fluxb_moe_permute", "fluxb_moe_unpermute", "fluxb_moe_route"):
        assert seen[name] == bits(lazy)
    moe._RouteFn.backward(_Context((index, torch.ones(1, 1)), like=(torch.float32, 8)), None, lazy)
    rows = torch.ones(1, 1)
    moe._UnpermuteFn.backward(_Context((rows, splits, index, rows), like=(torch.float32, 1), needs_input_grad=(True, False, False, True)), lazy)
    for name in ("fluxb_moe_route_backward", "fluxb_moe_unpermute_backward"):
        assert seen[name] == bits(lazy)


@pytest.mark.parametrize("dtype,size", [(_lib.F32, 4), (_lib.BF16, 2), (_lib.F16, 2)])
def test_addresses_off_their_type_are_refused(dtype, size):
    """A load or store across its type's boundary is a fault of the GPU: such addresses do not reach it."""
    lib = _lib.load()
    at = lambda p: C.c_void_p(p)  # noqa: E731
    good = 256

    def refused(rc, who):
        assert rc == _lib.FLUXB_ERR_INVALID and who in _lib.last_error() and "aligned" in _lib.last_error()

    def each(call, who, sizes):
        """Every pointer in turn one byte, and half of its type, off."""
        for i, n in enumerate(sizes):
            for off in {1, n // 2}:
                if off < n:
                    p = [at(good)] * len(sizes)
                    p[i] = at(good + off)
                    if off:
                        refused(call(*p), who)

    each(lambda z, c, w: lib.fluxb_moe_route(z, dtype, 4, 8, 2, c, w, None), "moe_route", (size, 4, 4))
    each(lambda dw, c, w, dz: lib.fluxb_moe_route_backward(dw, c, w, dtype, 4, 8, 2, dz, None), "moe_route_backward", (4, 4, 4, size))
    each(lambda x, s, i, r: lib.fluxb_moe_permute(x, 4, 2, 7, s, 8, i, r, None), "moe_permute", (1, 4, 4, 1))
    each(lambda r, i, w, o: lib.fluxb_moe_unpermute(r, dtype, 4, 2, 7, i, w, dtype, o, None), "moe_unpermute", (size, 4, size, size))
    each(lambda do, r, s, i, w, dr, dw: lib.fluxb_moe_unpermute_backward(do, r, dtype, 4, 2, 7, s, 8, i, w, dtype, dr, dw, None), "moe_unpermute_backward",
         (size, size, 4, 4, size, size, size))
    each(lambda s, i: lib.fluxb_mx_quantize(at(256), dtype, 1, 4, 32, 32, at(256), at(256), s, 8, i, 2, None), "mx_quantize", (4, 4))
    each(lambda s: lib.fluxb_mx_grouped_gemm(at(256), at(256), at(256), 4, at(256), at(256), 2, s, at(256), 8, 32, dtype, at(256), None, None),
         "mx_grouped_gemm", (4,))
