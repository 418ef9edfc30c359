"""The text decoder's program on the CPU, with a model that only takes down what it is asked."""
import pytest
import torch

from kitchen_amd import generate


class Recorder:
    """In the decoder's place: logits without a number for every second sequence, and the tokens of every step."""
    steps = []

    def __init__(self, config, seqs, *args, **kw):
        self.config, self.seqs, self.cache = config, seqs, self
        Recorder.steps = []

    def prompt(self, prompts):
        return torch.randn((len(prompts), self.config.vocab))

    def step(self, tokens, rows):
        Recorder.steps.append(tokens.clone())
        logits = torch.randn((self.seqs, self.config.vocab))
        logits[::2] = float("nan")
        return logits

    def check(self):
        pass

    def fork(self, src, dst):
        pass

    def free(self, rows):
        pass

    def compact(self):
        return torch.ones(1, dtype=torch.int32)


@pytest.mark.parametrize("temperature", ["0", "0.8"])
def test_tokens_of_rows_without_a_number_are_in_the_table(monkeypatch, capsys, temperature):
    """sample says -1 for a row of NaNs; an embedding has no such row (on the device the lookup would end the process)."""
    from oracle import step

    def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        return torch.tensor([step.sample(x.numpy(), float(y), temperature, top_k, top_p, min_p) for x, y in zip(logits, u)])

    monkeypatch.setattr(generate, "Decoder", Recorder)
    monkeypatch.setattr(generate.step, "sample", sample)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    assert generate.main(["--prompts", "2", "--alternatives", "2", "--tokens", "3", "--length", "8", "--temperature", temperature]) == 0
    assert len(Recorder.steps) == 3 and "3 steps in" in capsys.readouterr().out
    for tokens in Recorder.steps:
        assert int(tokens.min()) >= 0 and int(tokens.max()) < generate.Config.vocab
    assert all((tokens[::2] == 0).all() for tokens in Recorder.steps[1:])


@pytest.mark.parametrize("int8", [False, True])
def test_no_plan_where_none_can_pay(monkeypatch, int8):
    """The most that a plan can save is every row but one reading all pages that a row or the cache has; a step asks for a plan
    only where that is as much as a plan has to save."""
    from types import SimpleNamespace

    from kitchen_amd import kv

    # 4 heads of 128, keys and values: 2048 (int8: 1024) bytes a token; 20 pages of 16 for 7 rows more: 320 * 7 tokens
    cache = kv.PagedKVCache(1, 20, 4, 128, 16, 8, 1000, int8=int8, device="cpu")
    most = 320 * 7 * (1024 if int8 else 2048)
    plans = []
    monkeypatch.setattr(cache, "grow", lambda rows, counts: None)
    monkeypatch.setattr(cache, "shared", lambda lens: plans.append(1) or "plan")
    model = SimpleNamespace(cache=cache, _forward=lambda tokens, cu_q, lens, shared: shared, _logits=lambda x: x)
    rows = torch.arange(8)

    def step(least):
        monkeypatch.setattr(kv, "LEAST_SHARED", least)
        return generate.Decoder.step(model, rows, rows)

    assert [step(least) for least in (0, most, 1 << 40)] == [None] * 3          # nothing has forked
    cache.forked = True
    assert [step(least) for least in (0, most, most + 1, 100 << 20)] == ["plan", "plan", None, None]
    assert len(plans) == 2
    assert cache.may_share(most) and not cache.may_share(most + 1)
