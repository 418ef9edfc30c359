"""The small decoder (kitchen_amd.generate): what it computes over its paged cache, prompt by prompt and token by
token, against the same network in fp32 without a cache on the dequantized weights.

Tolerance: with floating activations everywhere the only roundings are bf16 ones (2^-9 relative each) of some ten
tensors per layer that a residual adds up: with L layers a relative distance of about sqrt(10 L) 2^-9, 1.2 % for
three; 4 % is allowed. An int8 cache rounds keys and values by up to absmax / 254 per value (0.5 % of a head's norm
for normal values): 6 %. int8 activations (a prompt's linears) round by absmax / 254 of a rotated row, about 0.8 % per
linear, 4 a layer, 3 layers: 2.7 % more, 8 %."""
import pytest
import torch

from kitchen_amd import comfy_formats, generate


def plain(model, tokens):
    """Logits behind every token, fp32."""
    c = model.config

    def linear(layer, x):
        w = comfy_formats.dequantize_w4a8(layer.q, layer.s, layer.z, layer.GROUP, layer.ROTATE, torch.float32)
        return x @ w.t()

    n = len(tokens)
    pos = torch.arange(n, device=tokens.device)
    x = model.embedding[tokens].float() * c.hidden ** 0.5
    for i, layer in enumerate(model.layers):
        q, k, v = linear(layer["qkv"], generate._norm(x)).view(n, -1, c.head_dim).split([c.heads, c.kv_heads, c.kv_heads], 1)
        q, k = generate._turn(q, pos), generate._turn(k, pos)
        seen = pos[None] <= pos[:, None]
        if c.window and i % 2:
            seen &= (pos[:, None] - pos[None] < c.window) | (pos[None] < c.sinks)
        out = []
        for h in range(c.heads):
            g = h // (c.heads // c.kv_heads)
            a = (q[:, h] @ k[:, g].t() * c.head_dim ** -0.5).masked_fill(~seen, float("-inf"))
            out.append(torch.softmax(a, -1) @ v[:, g])
        x = x + linear(layer["out"], torch.stack(out, 1).view(n, -1))
        gate, up = linear(layer["up"], generate._norm(x)).chunk(2, -1)
        x = x + linear(layer["down"], torch.nn.functional.silu(gate) * up)
    return generate._norm(x) @ model.embedding.float().t()


def distance(y, want):
    return ((y.float() - want).norm() / want.norm()).item()


def small(**kw):
    c = dict(layers=3, hidden=512, heads=8, kv_heads=2, head_dim=64, inner=768, vocab=320)
    return generate.Config(**dict(c, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("window,int8,few,tol", [(None, False, 1 << 30, 0.04), (24, False, 1 << 30, 0.04),
                                                 (None, True, 1 << 30, 0.06), (40, False, 16, 0.08)])
def test_decoder(gpu_device, window, int8, few, tol):
    print(f"[generate] window {window} int8 {int8} few {few}", flush=True)
    model = generate.Decoder(small(window=window, sinks=3 if window else 0), seqs=5, pages=64, max_tokens=128, int8_cache=int8, few=few)
    g = torch.Generator().manual_seed(3)
    text = [torch.randint(320, (n,), generator=g).tolist() for n in (70, 1, 33)]
    # prompts in sequences 0, 1 and 3, the first one in two chunks
    first = model.prompt({0: text[0][:50], 1: text[1]})
    second = model.prompt({0: text[0][50:], 3: text[2]})
    model.cache.check()
    dev = gpu_device
    ref = [plain(model, torch.tensor(t, device=dev)) for t in text]
    assert distance(first[0], ref[0][49]) < tol and distance(first[1], ref[1][0]) < tol
    assert distance(second[0], ref[0][69]) < tol and distance(second[1], ref[2][32]) < tol
    # sequence 2 becomes an alternative of 0, 4 of 3; all go on with tokens of their own
    model.cache.fork([0, 3], [2, 4])
    model.cache.check()
    text = {0: text[0], 1: text[1], 2: text[0], 3: text[2], 4: text[2]}
    rows = list(text)
    for n in range(12):
        if n == 6:                                    # 1 and 4 end, the pages of the others move together
            model.cache.free([1, 4])
            held = int(model.cache.compact())
            assert held == int((model.cache.refs > 0).sum()) and (model.cache.refs[:held] > 0).all()
            rows = [0, 2, 3]
        new = torch.randint(320, (5,), generator=g)
        y = model.step(new.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev))
        text = {b: text[b] + [int(new[b])] for b in rows}
    model.cache.check()
    for b in rows:
        assert distance(y[b], plain(model, torch.tensor(text[b], device=dev))[-1]) < tol, b
    assert model.cache.lens.tolist() == [82, 0, 82, 45, 0]


@pytest.mark.gpu
def test_command(gpu_device, capsys):
    assert generate.main(["--prompts", "2", "--length", "40", "--tokens", "6", "--layers", "2", "--window", "16", "--int8-cache"]) == 0
    out = capsys.readouterr().out
    assert "prompt 1, alternative 1:" in out and "6 steps in" in out


@pytest.mark.gpu
def test_cache_too_small(gpu_device):
    model = generate.Decoder(small(), seqs=2, pages=3, max_tokens=128)
    model.prompt({0: [1] * 60})
    with pytest.raises(Exception, match="1 pages short"):
        model.cache.check()
    assert model.cache.lens.tolist() == [0, 0]
