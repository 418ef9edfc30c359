"""The small decoder at the sizes of its command. Tolerance as in test_gpu_generate.py."""
import pytest
import torch

from kitchen_amd import generate
from test_gpu_generate import distance, plain


@pytest.mark.gpu
def test_a_batch_at_the_programs_sizes(gpu_device):
    """The program's own configuration (hidden 2048, 8 sequences: linears of several column tiles a workgroup) against
    the fp32 network, token by token. The tolerance of test_gpu_generate.py for floating activations: 4 %."""
    print("[generate] the program's sizes", flush=True)
    model = generate.Decoder(generate.Config(layers=2, vocab=512), seqs=8, pages=64, max_tokens=64)
    g = torch.Generator().manual_seed(7)
    texts = {b: torch.randint(512, (3 + b,), generator=g).tolist() for b in range(8)}
    model.prompt({b: t[:-1] for b, t in texts.items()})
    rows = torch.arange(8, dtype=torch.int32, device=gpu_device)
    y = model.step(torch.tensor([t[-1] for t in texts.values()], device=gpu_device), rows)
    model.cache.check()
    for b, t in texts.items():
        assert distance(y[b], plain(model, torch.tensor(t, device=gpu_device))[-1]) < 0.04, b
