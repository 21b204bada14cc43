"""Communicators made by several threads at once: one per group, and none is released while a caller holds its handle. The native
communicator is a stand-in; nothing here needs a GPU."""
import threading
import time

import pytest

from flux_b200 import mx, shm


class _Comm:
    made = []

    def __init__(self, group):
        time.sleep(0.05)  # (the native call and the barrier let other threads run)
        self.group, self.handle = group, object()
        self.device = type("", (), {"index": 0})
        _Comm.made.append(self)


@pytest.fixture(autouse=True)
def nothing_made_yet(monkeypatch):
    _Comm.made = []
    monkeypatch.setattr(shm, "Comm", _Comm)
    monkeypatch.setattr(shm, "_COMMS", {})
    monkeypatch.setattr(mx, "Comm", _Comm)
    monkeypatch.setattr(mx, "_COMMS", {})
    monkeypatch.setattr(mx, "_USED", {}, raising=False)
    monkeypatch.setattr(mx, "_cur_device", lambda: 0)
    last = list(shm._LAST)
    shm._LAST.clear()
    yield
    shm._LAST[:] = last


def _together(call, n=6):
    start, got = threading.Barrier(n), [None] * n

    def work(i):
        start.wait()
        got[i] = call(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


def test_one_group_has_one_communicator():
    for group in (None, object()):
        got = _together(lambda i: shm.get_comm(group))
        assert len(set(map(id, got))) == 1 and shm.default_comm() is got[0]
    assert len(_Comm.made) == 2


def test_groups_do_not_wait_for_each_other():
    """Setting a communicator up is a collective of its group: two groups whose ranks begin in different orders must not block."""
    groups = [object(), object()]
    meet = threading.Barrier(2, timeout=10)

    class Collective(_Comm):
        def __init__(self, group):
            meet.wait()  # both are being made at the same time
            super().__init__(group)

    shm.Comm = Collective  # (put back by the fixture)
    got = _together(lambda i: shm.get_comm(groups[i]), 2)
    assert [c.group for c in got] == groups


def test_first_products_share_a_communicator():
    got = _together(lambda i: mx._comm())
    assert len(set(map(id, got))) == 1 and len(_Comm.made) == 1


def test_first_products_beside_a_default_of_another_device():
    shm.get_comm(None).device = type("", (), {"index": 1})
    got = _together(lambda i: mx._comm())
    assert len(set(map(id, got))) == 1 and len(_Comm.made) == 2 and got[0] is not shm.default_comm()


def test_products_do_not_make_a_default_communicator():
    """Ops that bind to the communicator of `init_flux_shm` still ask for it."""
    c = mx._comm()
    with pytest.raises(RuntimeError, match="call flux.init_flux_shm"):
        shm.default_comm()
    assert mx._comm() is c and len(_Comm.made) == 1
    default = shm.get_comm(None)
    assert default is not c and mx._comm() is default


def _with_status(c, status):
    def check_status():
        if status:
            raise RuntimeError(f"status {status}")

    c.check_status = check_status
    return c


def test_the_status_of_products_can_be_read():
    """Of every communicator that products of the current device have used, whichever is the default by now; of no other device's."""
    mx.mx_check_status()  # no product yet
    own = _with_status(mx._comm(), 0)
    default = _with_status(shm.get_comm(None), 0)
    mx._comm()
    later = _with_status(shm.get_comm(object()), 0)
    mx.mx_check_status()
    for c, used in ((own, True), (default, True), (later, False)):
        _with_status(c, 3)
        if used:
            with pytest.raises(RuntimeError, match="status 3"):
                mx.mx_check_status()
        else:
            mx.mx_check_status()  # no product has used it
        _with_status(c, 0)
    mx._cur_device = lambda: 1  # (put back by the fixture)
    _with_status(own, 3)
    mx.mx_check_status()
    other = _with_status(mx._comm(), 4)
    assert other not in (own, default, later)
    with pytest.raises(RuntimeError, match="status 4"):
        mx.mx_check_status()
