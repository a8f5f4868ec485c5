"""GPT-2 over the paged cache: the last rows of several sequences with different numbers of new tokens."""
import numpy as np
import pytest
import torch

from test_generation_model_gpu import CFG, close, reference, rounding, setup  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,page_size", [(None, 16), (torch.int8, 32)])
def test_the_last_row_of_each_sequence(setup, dtype, page_size):  # noqa: F811
    w, model = setup
    rng = np.random.default_rng(11)
    total = [120, 40, 9]
    tokens = [rng.integers(0, CFG.vocab_size, n).tolist() for n in total]
    want = [reference(w, t) for t in tokens]
    more = max(rounding(w, t, dtype) for t in tokens)
    c = model.new_cache(400, page_size, dtype)
    seqs = [c.open() for _ in total]
    done = [0, 0, 0]
    for step in ([100, 30, 5], [2, 1, 0], [1, 7, 1], [0, 1, 1], [17, 1, 2]):
        live = [b for b in (2, 0, 1) if step[b]]
        plan = c.extend([seqs[b] for b in live], [step[b] for b in live])
        ids = torch.tensor([t for b in live for t in tokens[b][done[b]:done[b] + step[b]]], dtype=torch.int32, device="cuda")
        last = model.forward_cached(ids, c, plan)
        done = [d + n for d, n in zip(done, step)]
        close(last, torch.stack([want[b][done[b] - 1] for b in live]), f"step {step}", more)
    # beside a sequence without a new token every row is still to be had
    plan = c.extend(seqs, [0, 0, 0])
    with pytest.raises(ValueError, match="no last row"):
        model.forward_cached(torch.zeros(0, dtype=torch.int32, device="cuda"), c, plan)
    rows = c.read(0, [seqs[1]], out_dtype=torch.float16)[0]
    assert rows.shape == (total[1], CFG.n_head, 64)
