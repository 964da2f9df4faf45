"""Adapters on the host: their checks, the engine's names, slots and graph keys,
and the dispatcher that keeps every GPU's set, with fakes of the native engine."""
import queue
import threading
import time
import types

import numpy as np
import pytest

from laya_b200.config import TINY
from laya_b200.dispatcher import B200Dispatcher
from laya_b200.engine import B200Engine, _Lane, request_from_items
from laya_b200.weights import adapted_projections, bf16_bits_to_f32, check_adapter

D, I = TINY.hidden, TINY.intermediate


def adapter(rank=4, names=("enc.0.wqkv",), fill=0.5):
    shapes = adapted_projections(TINY)
    return {n: (np.full((rank, shapes[n][1]), fill, np.float32), np.ones((shapes[n][0], rank), np.float32))
            for n in names}


def test_projections_and_conversion():
    shapes = adapted_projections(TINY)
    assert len(shapes) == 4 * TINY.layers
    assert shapes["enc.2.wi"] == (2 * I, D) and shapes["enc.0.wo2"] == (D, I)
    got = check_adapter(adapter(fill=1.00390625), TINY)  # half a bf16 step above 1: to even
    a, b = got["enc.0.wqkv"]
    assert a.dtype == b.dtype == np.uint16 and (bf16_bits_to_f32(a) == 1.0).all()
    again = check_adapter(got, TINY)["enc.0.wqkv"]
    assert np.array_equal(again[0], a) and np.array_equal(again[1], b)


def bad_adapters():
    ok = adapter()["enc.0.wqkv"]
    inf = ok[0].copy()
    inf[1, 2] = np.inf
    big = ok[0].copy()
    big[0, 0] = 3.4e38  # rounds to infinity in bf16
    bits = np.full(ok[0].shape, 0x7FC0, np.uint16)
    return [{}, {"enc.9.wqkv": ok}, {"embed.tok": ok}, {"head.0.in_proj.w": ok}, {"enc.0.wo": ok},
            {"enc.0.wqkv": (ok[0].T, ok[1])}, {"enc.0.wqkv": (ok[0], ok[1][:, :3])}, {"enc.0.wqkv": (inf, ok[1])},
            {"enc.0.wqkv": (big, ok[1])}, {"enc.0.wqkv": (bits, ok[1])}, {"enc.0.wqkv": (ok[0].astype(int), ok[1])},
            {"enc.0.wqkv": (ok[0][:0], ok[1][:, :0])}]


@pytest.mark.parametrize("bad", bad_adapters())
def test_bad_adapters_are_refused(bad):
    with pytest.raises(ValueError):
        check_adapter(bad, TINY)


def test_rank_limit():
    check_adapter(adapter(rank=16), TINY, 16)
    with pytest.raises(ValueError):
        check_adapter(adapter(rank=17), TINY, 16)


class FakeNative:
    def __init__(self):
        self.captured, self.runs, self.slots, self.fail = [], [], {}, False

    def capture(self, *key):
        self.captured.append(("plain", *key))
        return len(self.captured) - 1

    def capture_adapters(self, *key):
        self.captured.append(("adapters", *key))
        return len(self.captured) - 1

    def release(self, slot):
        pass

    def run(self, slot, inputs, adapter=None):
        self.runs.append(None if adapter is None else adapter.tolist())
        b, k = inputs["marker_pos"].shape
        return np.zeros((b, k), np.float32), np.zeros((b, 2), np.float32)

    def set_adapter(self, slot, adapter, scaling):
        if self.fail:
            raise RuntimeError("upload failed")
        self.slots[slot] = scaling

    def clear_adapter(self, slot):
        self.slots.pop(slot, None)

    def close(self):
        pass


def engine(slots=2, lanes=1):
    e = B200Engine.__new__(B200Engine)
    from collections import OrderedDict
    e.lock, e.max_questions, e.max_graphs = threading.RLock(), 64, 8
    e.sequence_buckets, e.cfg, e.pad_token_id, e.max_options = (64, 128), {"max_len": 128}, 0, 16
    e.backend, e.precision, e.device = "b200-bf16", "bf16", 0
    e.graphs, e.closed, e.config = OrderedDict(), False, TINY
    e.native = FakeNative()
    e.adapter_rank, e.adapters, e._free_adapters = 8, {}, list(range(slots))
    e._lanes = [e] + [_Lane(FakeNative()) for _ in range(lanes - 1)]
    e._idle = queue.Queue()
    for lane in e._lanes:
        e._idle.put(lane)
    return e


def request(*names):
    return request_from_items([{"ids": [1] * 64, "markers": [1, 2], "qtype": 0, **({"adapter": n} if n else {})}
                               for n in names])


def test_questions_select_adapters_by_name():
    e = engine()
    e.load_adapter("a", adapter(), 2.0)
    e.load_adapter("b", adapter())
    assert e.native.slots == {0: 2.0, 1: 1.0}
    e.run_prepared(request("b", None, "a"))
    e.run_prepared(request(None, None))       # no question has one: the plain graph
    e.run_prepared(request("b", "b", "a"))    # the same graph again
    assert e.native.runs == [[1, -1, 0, -1], None, [1, 1, 0, -1]]
    assert [c[0] for c in e.native.captured] == ["adapters", "plain"]
    assert e._graph_key(request("a", "a")) != e._graph_key(request(None, None))


def test_slots_are_reused_and_errors_leave_the_engine_usable():
    e = engine()
    e.load_adapter("a", adapter())
    e.load_adapter("b", adapter())
    with pytest.raises(RuntimeError, match="no adapter slot"):
        e.load_adapter("c", adapter())
    e.load_adapter("b", adapter(), 3.0)       # replaces in its own slot
    assert e.adapters == {"a": 0, "b": 1} and e.native.slots[1] == 3.0
    e.unload_adapter("a")
    assert 0 not in e.native.slots
    e.load_adapter("c", adapter())
    assert e.adapters == {"b": 1, "c": 0}
    for bad in (("x", {}), (None, adapter()), ("x", adapter(rank=9))):
        with pytest.raises(ValueError):
            e.load_adapter(*bad)
    with pytest.raises(ValueError):
        e.load_adapter("x", adapter(), float("nan"))
    with pytest.raises(ValueError):
        e.unload_adapter("a")
    with pytest.raises(ValueError, match="no adapter 'a'"):
        e.run_prepared(request("a"))
    e.native.fail = True
    with pytest.raises(RuntimeError, match="upload"):
        e.load_adapter("c", adapter())
    assert e.adapters == {"b": 1} and e._free_adapters == [0]
    e.native.fail = False
    e.load_adapter("d", adapter())
    e.run_prepared(request("d"))
    assert e.native.runs == [[0]]
    e.closed = True
    with pytest.raises(RuntimeError, match="closed"):
        e.load_adapter("e", adapter())


def test_loading_waits_for_every_lane():
    e = engine(lanes=2)
    busy = e._idle.get()
    done = threading.Event()
    t = threading.Thread(target=lambda: (e.load_adapter("a", adapter()), done.set()))
    t.start()
    assert not done.wait(0.1) and e.adapters == {}
    e._idle.put(busy)
    assert done.wait(5)
    t.join()
    assert e._idle.qsize() == 2 and e.adapters == {"a": 0}


def test_constructor_checks():
    for kw in (dict(adapters=-1), dict(adapters=1, adapter_rank=0), dict(adapters=1, adapter_rank=257),
               dict(adapters=1, precision="nvfp4")):
        with pytest.raises(ValueError):
            B200Engine(config=TINY, **kw)


# ---------------------------------------------------------------- dispatcher
class FakeEngine:
    def __init__(self, device, fail_load=()):
        self.device, self.adapters, self.fail_load, self.fail = device, {}, set(fail_load), False
        self.delay = 0.0

    def load_adapter(self, name, adapter, scaling=1.0):
        if name in self.fail_load:
            raise RuntimeError("no adapter slot is free")
        self.adapters[name] = scaling

    def unload_adapter(self, name):
        del self.adapters[name]

    def run_prepared(self, prepared):
        time.sleep(self.delay)
        if self.fail:
            raise RuntimeError("injected")
        for it in prepared.items:
            assert it.get("adapter") in (None, *self.adapters)
        n = len(prepared.items)
        return np.zeros((n, 2), np.float32), np.zeros((n, 2), np.float32), {}

    def close(self):
        pass


def dispatcher(**fail):
    engines = {}

    def factory(device, **_):
        engines[device] = FakeEngine(device, fail.get(f"gpu{device}", ()))
        return engines[device]

    return B200Dispatcher(devices=[0, 1], engine_factory=factory), engines


def items(*names):
    return [{"ids": [1] * (40 + 64 * i), "markers": [1, 2], "qtype": 0, "adapter": n} for i, n in enumerate(names)]


def test_dispatcher_keeps_every_gpu_alike():
    d, e = dispatcher(gpu1=["bad"])
    with d:
        d.load_adapter("a", adapter(), 2.0)
        assert e[0].adapters == e[1].adapters == {"a": 2.0}
        with pytest.raises(RuntimeError, match="slot"):
            d.load_adapter("bad", adapter())
        assert e[0].adapters == e[1].adapters == {"a": 2.0} and all(d.healthy.values())
        assert len(d.run_items(items("a", None, "a", None))) == 4
        with pytest.raises(ValueError, match="no adapter"):
            d.run_items(items("a", "b"))
        assert all(d.healthy.values())  # the caller's error takes no GPU out of service
        d.unload_adapter("a")
        assert e[0].adapters == e[1].adapters == {}
        with pytest.raises(ValueError):
            d.unload_adapter("a")
        with pytest.raises(ValueError):
            d.run_items(items("a"))


def test_a_readmitted_gpu_gets_what_it_missed():
    d, e = dispatcher()
    with d:
        d.load_adapter("old", adapter())
        e[1].fail = True
        d.run_items(items("old", None, "old", None))
        assert d.healthy == {0: True, 1: False}
        d.load_adapter("new", adapter())
        d.unload_adapter("old")
        assert e[1].adapters == {"old": 1.0}
        e[1].fail = False
        assert d.readmit(items(None)) == [1]
        assert e[0].adapters == e[1].adapters == {"new": 1.0}
        d.run_items(items("new", "new", "new", "new"))
        assert all(d.healthy.values())


def test_adapters_change_between_requests_only():
    d, e = dispatcher()
    with d:
        d.load_adapter("a", adapter())
        for x in e.values():
            x.delay = 0.2
        out = []
        t = threading.Thread(target=lambda: out.append(d.run_items(items("a", "a", "a", "a"))))
        t.start()
        time.sleep(0.05)
        d.unload_adapter("a")  # waits for the request, whose workers check that it is still loaded
        t.join()
        assert len(out) == 1 and all(d.healthy.values()) and e[0].adapters == {}


def test_adapter_unloaded_between_check_and_run():
    """The slots are looked up again when a lane takes the request."""
    engine = B200Engine.__new__(B200Engine)
    engine.adapters = {"a": 3}
    prepared = types.SimpleNamespace(items=[{"adapter": "a"}, {}, {"adapter": None}])
    assert engine._adapter_slots(prepared, 4).tolist() == [3, -1, -1, -1]
    del engine.adapters["a"]
    with pytest.raises(ValueError, match="no adapter 'a'"):
        engine._adapter_slots(prepared, 4)
