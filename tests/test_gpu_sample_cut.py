"""sample's top_p where it cuts next to the end of thousands of equal values, against the plain choice in 64 bits."""
import numpy as np
import pytest
import torch

import kitchen_amd as ck
from oracle import step

# A best value of 0, n equal ones that top_p cuts, m below those and one between that makes their weights meet: half of all weight
# ends 3e-8 (of the n values' weight; 2e-7 in the longest row) in front of the end of the n values, so all of them are kept and
# nothing below. 1 / n of their weight is 8e-5 (5e-6): the margin on the other side. Sums of bins and of single weights that differ
# by more than the first would keep the whole row.
NEXT_TO_THE_END = [(100000, -9.918127059936523, 12000, -10.418127059936523, 53244, -10.111069679260254),
                   (131072, -9.918127059936523, 12000, -10.418127059936523, 53244, -10.111069679260254),
                   (200000, -9.918127059936523, 12000, -10.418127059936523, 53244, -10.111085891723633),
                   (1 << 20, -11.925908088684082, 200000, -12.425908088684082, 578917, -12.068163871765137)]


def row(vocab, v, n, below, m, between):
    x = np.full(vocab, -np.inf, dtype=np.float32)
    x[:m] = below
    x[m] = between
    x[m + 1] = 0.0
    x[vocab - n:] = v
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("case", NEXT_TO_THE_END, ids=lambda c: str(c[0]))
@pytest.mark.parametrize("rows", [1, 300])
def test_a_cut_next_to_the_end_of_thousands_alike(gpu_device, case, rows):
    if rows * case[0] > 1 << 26:
        rows = 260                                      # (more than the compute units, as 300)
    x = row(*case)
    w = np.exp(x.astype(np.float64))
    share = (w.sum() / 2 - w[x >= case[1]].sum()) / w[x == np.float32(case[1])].sum()
    assert -1e-6 < share < -1e-8                        # as the comment above says
    u = np.linspace(0.01, 0.99, 9).astype(np.float32)
    want = [step.sample(x, y, top_p=0.5) for y in u]
    assert min(want) > case[4]                          # nothing of what lies below
    logits = torch.from_numpy(x).to(gpu_device).expand(rows, -1)
    logits = logits if rows == 1 else logits.contiguous()
    for y, t in zip(u, want):
        got = ck.sample(logits, torch.full((rows,), float(y), device=gpu_device), top_p=0.5)
        assert got.tolist() == [t] * rows


@pytest.mark.gpu
@pytest.mark.parametrize("v", [-15.03, -15.71, -16.22, -16.64, -17.05, -17.4])
@pytest.mark.parametrize("rows", [1, 300])
def test_tokens_among_small_weights(gpu_device, v, rows):
    """A best value (weight 1) and n = 131071 equal ones of weight w = 2^-25.1 to 2^-21.7 behind it: where token i is chosen, u lies
    (1 - u) / w = n - i weights in front of the end of all of them. A weight off by 2e-9 of itself and a unit (2^-45) moves that
    place by (n - i) (2e-9 + 2^-45 / w) <= 0.14 tokens at w = 2^-25.1, so a place in the middle third of a token stays in it."""
    vocab = 1 << 17
    x = np.full(vocab, np.float32(v), dtype=np.float32)
    x[0] = 0.0
    w, n = float(np.exp(np.float64(x[1]))), vocab - 1
    us = []
    for i in (3, 70, 1000, 20000, 65536, 100000, 131000):
        u = np.float32((1 + (i + 0.5) * w) / (1 + n * w))
        for _ in range(64):                             # the next one whose place is in the middle third
            at = (float(u) * (1 + n * w) - 1) / w
            if 1 / 3 < at % 1 < 2 / 3 and 0 < at < n:
                us.append((u, 1 + int(at)))
                break
            u = np.nextafter(u, np.float32(0 if i == 131000 else 2))
    assert len(us) == 7
    logits = torch.from_numpy(x).to(gpu_device).expand(rows, -1)
    logits = logits if rows == 1 else logits.contiguous()
    for u, t in us:
        assert step.sample(x, u) == t                    # the oracle's sums of fp64 say the same
        assert ck.sample(logits, torch.full((rows,), float(u), device=gpu_device)).tolist() == [t] * rows, (float(u), t)
