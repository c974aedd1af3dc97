"""The serving loop of the paged example, without a GPU: a stub engine answers with numbers. Prompts that no step can
take are refused before the first one, and every loop that starts ends."""
import importlib.util
import sys

import pytest

from conftest import REPO


@pytest.fixture(scope="module")
def serving():
    pytest.importorskip("torch")
    if "paged_serving" not in sys.modules:
        spec = importlib.util.spec_from_file_location("paged_serving", REPO / "examples" / "paged_serving.py")
        sys.modules["paged_serving"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["paged_serving"])
    return sys.modules["paged_serving"]


class Stub:
    """An engine without a model: the id of a request is the number of tokens its row holds."""

    def __init__(self, rows, tokens, context):
        self.rows, self.tokens, self.context = rows, tokens, context
        self.held, self.counts, self.steps = [0] * rows, [[0, 0, 0, 0]], 0

    def plan(self, append):
        self.held = [0 if a < 0 else n + a for n, a in zip(self.held, append)]

    def step(self, append, ids, *controls):
        self.steps += 1
        assert self.steps < 1000, "the loop does not end"
        assert len(ids) == sum(max(0, a) for a in append) <= self.tokens
        self.plan(append)
        assert max(self.held) <= self.context
        stub = self

        class Out:
            def tolist(self):
                return list(stub.held)
        return Out()


@pytest.mark.parametrize("lengths,new_tokens,message", [
    ([3, 0, 4], 5, "prompt 1 is empty"), ([3, 29], 2, "prompt 1 has 29 ids"), ([500], 2, "prompt 0 has 500 ids"),
    ([4, 28], 14, "prompt 1 .*context"), ([4], 0, "new_tokens"), ([4], -3, "new_tokens")])
def test_prompts_that_no_step_can_take_are_refused(serving, lengths, new_tokens, message):
    engine = Stub(rows=4, tokens=32, context=40)
    with pytest.raises(ValueError, match=message):
        serving.serve(engine, [[1] * n for n in lengths], new_tokens)
    assert engine.steps == 0


@pytest.mark.parametrize("rows,tokens,context,lengths,new_tokens", [
    (4, 32, 40, [28, 1, 28, 3, 28, 28, 5, 28], 13), (1, 6, 20, [5, 5, 1], 16), (3, 40, 50, [1], 1), (2, 30, 31, [28] * 5, 4)])
def test_longest_prompts_are_served(serving, rows, tokens, context, lengths, new_tokens):
    engine = Stub(rows, tokens, context)
    answers = serving.serve(engine, [[1] * n for n in lengths], new_tokens)
    assert answers == [[n + i for i in range(new_tokens)] for n in lengths]
    assert engine.held == [0] * rows


def test_nothing_to_serve(serving):
    engine = Stub(2, 10, 10)
    assert serving.serve(engine, [], 3) == [] and engine.steps == 0
