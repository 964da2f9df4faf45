"""predict(), system_one() and warmup() with adapters, on the host: the tokeniser
and the native engine are fakes."""
import pytest

from laya_b200 import engine as engine_module
from laya_b200.protocol import PreparedRequest
from test_adapters_cpu import adapter, engine


@pytest.fixture
def served(monkeypatch):
    e = engine()
    e.tokenizer, e.temperature, e.temperature_by_options = object(), None, {}
    e.load_adapter("a", adapter())
    e.load_adapter("b", adapter())

    def prepare(self, state, questions):
        items = [{"ids": [1] * 64, "markers": [1, 2], "qtype": 0} for _ in questions]
        return PreparedRequest([q["id"] for q in questions], list(questions), items, 64 * len(items))

    monkeypatch.setattr(engine_module.B200Engine, "prepare", prepare)
    monkeypatch.setattr(engine_module, "format_response", lambda *_: {"answers": {}})
    return e


QUESTIONS = [{"id": "q0"}, {"id": "q1"}, {"id": "q2"}]


def test_questions_by_id(served):
    served.predict({}, QUESTIONS, adapters={"q0": "b", "q2": "a"})
    served.system_one({}, QUESTIONS, adapters="a")      # one for all
    served.warmup({}, QUESTIONS, adapters={"q1": None, "q0": "a"})
    served.predict({}, QUESTIONS)
    served.predict({}, QUESTIONS, adapters={})
    assert served.native.runs == [[1, -1, 0, -1], [0, 0, 0, -1], [0, -1, -1, -1], None, None]


@pytest.mark.parametrize("adapters, word", [({"q3": "a"}, "no question"), ({"q0": "c"}, "no adapter 'c'"),
                                            ("c", "no adapter 'c'")])
def test_refusals(served, adapters, word):
    with pytest.raises(ValueError, match=word):
        served.predict({}, QUESTIONS, adapters=adapters)
    assert served.native.runs == []
