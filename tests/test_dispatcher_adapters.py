"""Adapters in the dispatcher while GPUs leave and return to service, with fakes
of the engines."""
import threading

import numpy as np
import pytest

from laya_b200.dispatcher import B200Dispatcher


class Engine:
    """Adapters by name; load_adapter can be held up, and both calls fail on request."""

    def __init__(self):
        self.adapters, self.fail = {}, False
        self.hold = self.loading = None

    def load_adapter(self, name, adapter, scaling=1.0):
        if self.hold is not None:
            self.loading.set()
            assert self.hold.wait(10)
        if self.fail:
            raise RuntimeError("injected")
        self.adapters[name] = scaling

    def unload_adapter(self, name):
        del self.adapters[name]

    def run_prepared(self, prepared):
        if self.fail:
            raise RuntimeError("injected")
        for it in prepared.items:
            if it.get("adapter") not in (None, *self.adapters):
                raise ValueError(f"no adapter {it['adapter']!r} is loaded")
        n = len(prepared.items)
        return np.zeros((n, 2), np.float32), np.zeros((n, 2), np.float32), {}

    def close(self):
        pass


PAIR = {"enc.0.wqkv": (np.zeros((1, 2), np.float32), np.zeros((2, 1), np.float32))}


def items(*names):
    return [{"ids": [1] * (40 + 64 * i), "markers": [1, 2], "qtype": 0, "adapter": n} for i, n in enumerate(names)]


def dispatcher():
    engines = {}

    def factory(device, **_):
        engines[device] = Engine()
        return engines[device]

    return B200Dispatcher(devices=[0, 1], engine_factory=factory), engines


def drop_gpu_1(d, e):
    e[1].fail = True
    d.run_items(items(None, None, None, None))
    assert d.healthy == {0: True, 1: False}
    e[1].fail = False


@pytest.mark.parametrize("before", [[], ["old"]])
def test_readmitted_while_an_adapter_is_being_loaded(before):
    """A GPU that returns during another thread's load has that adapter too."""
    d, e = dispatcher()
    with d:
        for name in before:
            d.load_adapter(name, PAIR)
        drop_gpu_1(d, e)
        e[0].hold, e[0].loading = threading.Event(), threading.Event()
        load = threading.Thread(target=lambda: d.load_adapter("new", PAIR))
        load.start()
        assert e[0].loading.wait(10)
        back = []
        readmit = threading.Thread(target=lambda: back.extend(d.readmit(items(None))))
        readmit.start()
        readmit.join(0.3)  # it has probed, and found what there is to restore
        e[0].hold.set()
        load.join()
        readmit.join()
        assert back == [1] and all(d.healthy.values())
        assert e[0].adapters == e[1].adapters == dict.fromkeys([*before, "new"], 1.0)
        d.run_items(items("new", "new", "new", "new"))
        assert all(d.healthy.values())


def test_gpu_that_cannot_be_restored_stays_out():
    d, e = dispatcher()
    with d:
        d.load_adapter("a", PAIR)
        drop_gpu_1(d, e)
        d.load_adapter("b", PAIR)
        loads = e[1].load_adapter

        def refuse(name, *rest):
            if name == "b":
                raise RuntimeError("injected")
            loads(name, *rest)

        e[1].load_adapter = refuse
        assert d.readmit(items(None)) == [] and d.healthy == {0: True, 1: False}
        e[1].load_adapter = loads
        assert d.readmit(items(None)) == [1] and e[1].adapters == {"a": 1.0, "b": 1.0}


def test_readmit_does_not_wait_for_requests():
    d, e = dispatcher()
    with d:
        d.load_adapter("a", PAIR)
        drop_gpu_1(d, e)
        d.load_adapter("b", PAIR)
        go, started, run = threading.Event(), threading.Event(), e[0].run_prepared

        def slow(prepared):
            started.set()
            assert go.wait(10)
            return run(prepared)

        e[0].run_prepared = slow
        request = threading.Thread(target=lambda: d.run_items(items("a", "b")))
        request.start()
        assert started.wait(10)
        assert d.readmit(items(None)) == [1] and e[1].adapters == {"a": 1.0, "b": 1.0}
        go.set()
        request.join()
        assert all(d.healthy.values())


def test_probe_that_names_an_adapter():
    """A probe runs without adapters: those of the GPU are restored after it."""
    d, e = dispatcher()
    with d:
        drop_gpu_1(d, e)
        d.load_adapter("a", PAIR)
        probe = items("a")
        assert d.readmit(probe) == [1] and e[1].adapters == {"a": 1.0}
        assert probe == items("a")  # the caller's items are as they were


def test_load_without_a_healthy_gpu():
    """Nothing could check the adapter, and no GPU that it does not fit would return."""
    d, e = dispatcher()
    with d:
        d.load_adapter("a", PAIR, 2.0)
        e[0].fail = e[1].fail = True
        with pytest.raises(RuntimeError, match="no healthy GPU"):
            d.run_items(items(None, None, None, None))
        with pytest.raises(RuntimeError, match="no healthy GPU"):
            d.load_adapter("b", PAIR)
        with pytest.raises(RuntimeError, match="no healthy GPU"):
            d.load_adapter("a", PAIR, 3.0)
        e[0].fail = e[1].fail = False
        assert d.readmit(items(None)) == [0, 1]
        assert e[0].adapters == e[1].adapters == {"a": 2.0}
        d.unload_adapter("a")
        assert e[0].adapters == e[1].adapters == {}


@pytest.mark.parametrize("names", [("old", "new"), ("a", "b"), ("b", "a"), ("x", "y"), ("q1", "q0")])
def test_restored_with_every_slot_in_use(names):
    """What was unloaded meanwhile leaves its slot before the rest is loaded."""
    old, new = names
    d, e = dispatcher()
    for engine in e.values():
        loads = engine.load_adapter

        def limited(name, *rest, engine=engine, loads=loads):
            if name not in engine.adapters and len(engine.adapters) == 2:
                raise RuntimeError("no adapter slot is free")
            loads(name, *rest)

        engine.load_adapter = limited
    with d:
        d.load_adapter("kept", PAIR)
        d.load_adapter(old, PAIR)
        drop_gpu_1(d, e)
        d.unload_adapter(old)
        d.load_adapter(new, PAIR)
        assert d.readmit(items(None)) == [1] and e[1].adapters == e[0].adapters == {"kept": 1.0, new: 1.0}
