"""Plans in which a sequence has no new token, and steps with fewer rows than their plan."""
import pytest
import torch

from pequegrad_b200 import gpt2 as G
from test_generation_cpu import cache


def test_a_sequence_without_a_new_token_has_no_last_row():
    c = cache(8)
    a, b, d = c.open(), c.open(), c.open()
    c.extend([a, b, d], [5, 7, 3])
    p = c.extend([a, b, d], [0, 2, 0])
    assert p.last.tolist() == [-1, 1, -1] and p.fewest == 0 and p.rows == 2 and p.ctx_len.tolist() == [5, 9, 3]
    q = c.extend([b, a], [1, 4])
    assert q.last.tolist() == [0, 4] and q.fewest == 1
    model = G.GPT2.__new__(G.GPT2)  # refused before a weight is looked at
    model.cfg = G.GPT2Config(n_layer=2, n_head=3, n_embd=192, vocab_size=50, block_size=64)
    with pytest.raises(ValueError, match="no last row"):
        model.forward_cached(torch.zeros(2, dtype=torch.int32), c, p)
    assert c.extend([], []).fewest == 1  # a step of no sequences lacks no row


def test_a_step_with_fewer_rows_than_its_plan_is_refused():
    c = cache(8)
    p = c.extend([c.open()], [5])
    x = torch.zeros((4, 3, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="4 rows for a plan of 5"):
        c.write(0, x, x, p)
    with pytest.raises(ValueError, match="4 rows for a plan of 5"):
        c.attend(0, x, p)
