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
