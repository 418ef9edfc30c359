"""The small decoder with sequences that sit a step out, and with a cache that is too small: what sequences hold does
not change. Tolerance as in test_gpu_generate.py."""
import pytest
import torch

from test_gpu_generate import distance, plain, small
from kitchen_amd import generate


def _state(model):
    c = model.cache
    return [x.clone() for x in (c.k, c.v, c.page_table, c.lens, c.refs)]


@pytest.mark.gpu
@pytest.mark.parametrize("length", [37, 48])
def test_a_sequence_that_sits_out(gpu_device, length):
    """Sequences 0 and 1 (a fork of 0: at 48 tokens it shares every page) in turns, then together."""
    print(f"[generate] sits out {length}", flush=True)
    model = generate.Decoder(small(), seqs=3, pages=40, max_tokens=128, few=1 << 30)
    g = torch.Generator().manual_seed(3)
    text = torch.randint(320, (length,), generator=g).tolist()
    model.prompt({0: text})
    model.cache.fork([0], [1])
    model.cache.check()
    texts, dev = [list(text), list(text)], gpu_device

    def step(rows):
        new = torch.randint(320, (3,), generator=g)
        before = _state(model)
        y = model.step(new.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev))
        model.cache.check()
        for b in (0, 1):
            if b in rows:
                texts[b].append(int(new[b]))
            else:                                    # what it holds is as it was, in every layer
                pages = before[2][b][: -(-int(before[3][b]) // 16)].long()
                slots = int(before[3][b])
                for old, now in zip(before[:2], (model.cache.k, model.cache.v)):
                    was, now = (t[:, pages].transpose(2, 3).flatten(1, 2)[:, :slots] for t in (old, now))
                    assert torch.equal(was, now)
        return y

    for rows in ([0], [0], [1], [1], [1], [0], [1, 0]):
        y = step(rows)
    for b in (0, 1):
        assert distance(y[b], plain(model, torch.tensor(texts[b], device=dev))[-1]) < 0.04, b
    assert model.cache.lens.tolist() == [length + 4, length + 4, 0]


@pytest.mark.gpu
def test_a_step_without_room_changes_nothing(gpu_device):
    model = generate.Decoder(small(), seqs=2, pages=3, max_tokens=128)
    model.prompt({0: [1] * 32, 1: [2] * 16})
    model.cache.check()
    before = _state(model)
    model.step(torch.tensor([5, 6], device=gpu_device), torch.tensor([0, 1], dtype=torch.int32, device=gpu_device))
    with pytest.raises(Exception, match="2 pages short"):
        model.cache.check()
    assert all(torch.equal(a, b) for a, b in zip(before, _state(model)))
    model.prompt({1: [3, 4]})
    with pytest.raises(Exception, match="1 pages short"):
        model.cache.check()
    assert all(torch.equal(a, b) for a, b in zip(before, _state(model)))


@pytest.mark.gpu
def test_prompts_without_tokens_are_refused(gpu_device):
    model = generate.Decoder(small(layers=1), seqs=2, pages=3, max_tokens=128)
    for prompts in ({}, {0: [1, 2], 1: []}):
        with pytest.raises(ValueError, match="tokens"):
            model.prompt(prompts)
    assert not model.cache.lens.any()
