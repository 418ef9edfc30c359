"""The operators of a generation step one behind the other as generate.Decoder runs them: tokens of forks whose pages are read once
against the same step without the plan, and a captured step replayed against an eager one.

Tolerance of the first: both sides round the same tensors to bf16 in every layer, and a sum over keys in another order moves such
a rounding now and then; logits differ by at most what one such rounding in each of the two layers' tensors does,
2^-8 relative each, sqrt(2 x 10) of them: 1.8 %."""
import pytest
import torch

import kitchen_amd as ck
from kitchen_amd import generate


def small(**kw):
    c = dict(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, inner=768, vocab=320)
    return generate.Config(**dict(c, **kw))


def forked(config=None, int8=False, seed=0):
    """A decoder whose sequences 2 .. 5 are alternatives of 0 and 1."""
    model = generate.Decoder(config or small(), seqs=6, pages=120, max_tokens=256, int8_cache=int8, seed=seed)
    g = torch.Generator().manual_seed(seed)
    model.prompt({0: torch.randint(320, (100,), generator=g).tolist(), 1: torch.randint(320, (37,), generator=g).tolist()})
    model.cache.fork([0, 1, 0, 1], [2, 3, 4, 5])
    model.cache.check()
    return model


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [None, 24])
def test_forks_share_their_pages(gpu_device, monkeypatch, int8, window):
    print(f"[step] int8 {int8} window {window}", flush=True)
    monkeypatch.setattr(ck.kv, "LEAST_SHARED", 0)
    a, b = (forked(small(window=window, sinks=2 if window else 0), int8) for _ in range(2))
    b.cache.forked = False                          # this one reads every sequence's pages for itself
    plan = a.cache.shared().cpu().tolist()
    assert plan[0] == 2 and plan[4:10] == [96, 32] * 3
    rows = torch.arange(6, dtype=torch.int32, device=gpu_device)
    g = torch.Generator().manual_seed(5)
    for n in range(6):
        tokens = torch.randint(320, (6,), generator=g).to(gpu_device)
        if n == 3:                                  # the first sequences end: the others go on sharing
            for m in (a, b):
                m.cache.free([0, 1])
            rows = rows[2:]
            assert a.cache.shared().cpu().tolist()[4:10] == [0, 0, 96, 32, 96, 32]
        x, y = (m.step(tokens, rows)[rows.long()].float() for m in (a, b))
        assert (x - y).norm() < 0.018 * y.norm()


@pytest.mark.gpu
def test_sequences_that_sit_a_step_out(gpu_device):
    """Idle forks keep their pages; those that go on share them among themselves."""
    model = forked()
    before = model.cache.k.clone()
    rows = torch.tensor([2, 4, 5], dtype=torch.int32, device=gpu_device)
    model.step(torch.arange(6, device=gpu_device), rows)
    lens = model.cache.lens.tolist()
    assert lens == [100, 37, 101, 37, 101, 38]
    last = int(model.cache.page_table[0, 6])
    assert torch.equal(model.cache.k[:, last], before[:, last])


@pytest.mark.gpu
def test_a_step_in_a_graph(gpu_device, monkeypatch):
    """Growing, attending with a plan, sampling: captured once, replayed with other tokens and random numbers, against eager steps."""
    monkeypatch.setattr(ck.kv, "LEAST_SHARED", 0)
    a, b = forked(seed=3), forked(seed=3)
    rows = torch.arange(6, dtype=torch.int32, device=gpu_device)
    tokens, u = torch.zeros(6, dtype=torch.int64, device=gpu_device), torch.zeros(6, device=gpu_device)

    def step(model, tokens, u):
        return ck.sample(model.step(tokens, rows), u, temperature=0.9, top_k=40, top_p=0.95)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                   # a step of both before the capture
        for m in (a, b):
            step(m, tokens, u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, tokens, u)
    g = torch.Generator().manual_seed(6)
    for _ in range(5):
        tokens.copy_(torch.randint(320, (6,), generator=g))
        u.copy_(torch.rand(6, generator=g))
        graph.replay()
        want = step(b, tokens, u)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(a.cache.lens, b.cache.lens) and torch.equal(a.cache.k, b.cache.k) and torch.equal(a.cache.page_table, b.cache.page_table)


@pytest.mark.gpu
def test_command_with_sampling(gpu_device, capsys):
    args = ["--prompts", "2", "--length", "40", "--tokens", "8", "--layers", "2"]
    said = []
    # the model's output is its input's embedding again: a logit of 45 against normal ones, which a temperature of 0.8 does not
    # change and one of 60 does
    for more in ([], ["--temperature", "0.8", "--top-k", "50", "--top-p", "0.9", "--min-p", "0.01"], ["--temperature", "60"]):
        assert generate.main(args + more) == 0
        out = capsys.readouterr().out
        assert "prompt 1, alternative 1:" in out and "8 steps in" in out
        said.append([line for line in out.splitlines() if line.startswith("prompt ")])
    assert said[0] == said[1] != said[2]
