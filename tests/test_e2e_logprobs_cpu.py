"""What `e2e --logprobs` records, and what its timings hold, with a model and operators of the test's own."""
import types

import pytest
import torch

pytest.importorskip("transformers")


class Event:
    def __init__(self, enable_timing):
        pass

    def record(self):
        pass

    def elapsed_time(self, other):
        return 1.0


@pytest.fixture
def e2e(monkeypatch):
    from atflash import e2e
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    return e2e


VOCAB = 37


class Model:
    """Logits by the position; every call's are a tensor of its own, as a model's are."""
    config = None

    def __init__(self):
        self.at, self.given = 0, []

    def __call__(self, input_ids, past_key_values=None, use_cache=True, logits_to_keep=0):
        self.at += input_ids.shape[1]
        x = torch.randn((1, 1, VOCAB), generator=torch.Generator().manual_seed(self.at))
        self.given.append(x[:, -1].clone())
        return types.SimpleNamespace(logits=x)


@pytest.mark.parametrize("steps", [1, 6])
@pytest.mark.parametrize("top", [0, 3])
def test_logprobs_are_no_part_of_the_times(e2e, monkeypatch, steps, top):
    now = [0.0]
    monkeypatch.setattr(e2e.time, "perf_counter", lambda: now[0])

    def token_logprobs(logits, tokens, n):
        now[0] += 1000.0
        lp = torch.log_softmax(logits.double(), -1)
        vals, ids = lp.topk(n)
        return lp.gather(1, tokens[:, None])[:, 0], torch.special.entr(lp.exp()).sum(-1), vals, ids
    monkeypatch.setattr(e2e.ops, "token_logprobs", token_logprobs)
    hook = types.SimpleNamespace(new_cache=lambda *a: None)
    ids = torch.zeros((1, 10), dtype=torch.long)
    plain = e2e.run_request(Model(), hook, ids, 4, steps)
    model = Model()
    got = e2e.run_request(model, hook, ids, 4, steps, logprobs=top)
    said = got.pop("logprobs")
    assert "logprobs" not in plain and got == plain  # the times too
    assert len(said) == steps and got["wall_s"] == 0.0
    for tok, s, logits in zip(got["tokens"], said, model.given[-steps:]):
        lp = torch.log_softmax(logits.double(), -1)[0]
        assert tok == int(lp.argmax()) and s["logprob"] == pytest.approx(float(lp[tok]))
        assert s["entropy"] == pytest.approx(float(torch.special.entr(lp.exp()).sum()))
        assert len(s["top"]) == top and [i for i, _ in s["top"]] == lp.topk(top).indices.tolist()
        assert [x for _, x in s["top"]] == pytest.approx(lp.topk(top).values.tolist())
