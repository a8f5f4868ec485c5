"""The paged cache and the attention over it: strides, broadcast operands, queries that are no numbers, scales, captured chunks, threads."""
import pytest
import torch

from generation import Plan, new_cache
from pequegrad_b200 import kernels as K
from test_generation_gpu import attend, check, randn, same

pytestmark = pytest.mark.gpu

F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8

FORMS = [(F16, F16, 64, 4, 4), (BF16, BF16, 128, 8, 2), (F16, I8, 128, 6, 2), (BF16, I8, 64, 5, 1)]
STEPS = [([1, 3, 1], [700, 40, 130]), ([200, 30, 70], [700, 30, 300])]


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", FORMS)
@pytest.mark.parametrize("new,ctx", STEPS)
def test_padded_pitches_and_a_table_inside_a_larger_one(new, ctx, dtype, cache, D, Hq, Hkv):
    plan = Plan(new, ctx, 32)
    plain = new_cache(plan, Hkv, D, cache)
    pad = 16 if cache == I8 else 8

    def padded(x, n):  # the same values with room behind each run of the last dim
        y = torch.zeros((x.shape[0] + 1, x.shape[1], x.shape[2], x.shape[3] + n), dtype=x.dtype, device="cuda")[1:, ..., :x.shape[3]]
        return y.copy_(x)

    kc, vc = padded(plain[0], pad), padded(plain[1], 3 * pad)
    ks, vs = plain[2:] if cache != I8 else (torch.zeros((plan.pages, Hkv, 2, plan.P), device="cuda")[:, :, i].copy_(plain[2 + i]) for i in range(2))
    big = torch.full((len(new) + 2, plan.width + 7), 2 ** 30, dtype=torch.int32, device="cuda")
    big[1:-1, 3:3 + plan.width] = plan.table
    plan.table = big[1:-1, 3:3 + plan.width]
    q = randn(plan.rows, Hq + 1, D + 8, dtype=dtype)[:, 1:, :D]
    check(plan, attend(plan, q, (kc, vc, ks, vs)), q, plain)
    # and stored and read back through them
    x = randn(plan.rows, 2, Hkv, D, dtype=dtype if cache == I8 else cache, seed=2)
    other = [c.clone() for c in plain[:2]] + [c.clone() for c in plain[2:] if c is not None] + [None] * (2 if cache != I8 else 0)
    K.kv_write(x[:, 0], x[:, 1], kc, vc, plan.q_start, plan.ctx_len, plan.table, ks, vs)
    K.kv_write(x[:, 0], x[:, 1], other[0], other[1], plan.q_start, plan.ctx_len, plan.table.contiguous(), other[2], other[3])
    assert same(kc, other[0]) and same(vc, other[1])
    n = plan.kv_starts[-1]
    for a, b in zip(K.kv_read(kc, vc, plan.kv_start, plan.table, n, ks, vs), K.kv_read(other[0], other[1], plan.kv_start, plan.table, n, other[2], other[3])):
        assert same(a, b)


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", FORMS)
@pytest.mark.parametrize("new,ctx", STEPS)
def test_broadcast_operands_and_rows_before_the_first_sequence(new, ctx, dtype, cache, D, Hq, Hkv):
    plan = Plan(new, ctx, 32, pad_rows=2)
    c = new_cache(plan, Hkv, D, cache)
    # one query for all heads; one for all rows
    for q in (randn(plan.rows, 1, D, dtype=dtype).expand(-1, Hq, -1), randn(1, Hq, D, dtype=dtype).expand(plan.rows, -1, -1)):
        check(plan, attend(plan, q, c), q, c)
    # every page the same memory
    one = tuple(None if x is None else x[:1].expand(plan.pages, *x.shape[1:]) for x in c)
    q = randn(plan.rows, Hq, D, dtype=dtype)
    check(plan, attend(plan, q, one), q, one)
    # the first rows belong to nobody
    plan.q_start = plan.q_start + 3
    q = torch.cat([torch.full((3, Hq, D), float("nan"), dtype=dtype, device="cuda"), q])
    out = torch.full_like(q, 7)
    attend(plan, q, c, out=out)
    assert (out[:3] == 7).all() and (out[plan.starts[-1] + 3:] == 7).all()
    check(plan, out[3:], q[3:], c)


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", FORMS)
@pytest.mark.parametrize("new,ctx", STEPS)
def test_queries_that_are_not_numbers_spoil_their_rows_alone(new, ctx, dtype, cache, D, Hq, Hkv):
    plan = Plan(new, ctx, 32, pad_rows=5)
    c = new_cache(plan, Hkv, D, cache)
    q = randn(plan.rows, Hq, D, dtype=dtype)
    bad = q.clone()
    bad[1, 0, 3], bad[plan.starts[-1] - 1, Hq - 1, 0] = float("nan"), float("inf")
    bad[plan.starts[-1]:] = float("nan")  # padding
    n = plan.starts[-1]
    clean, got = attend(plan, q, c)[:n], attend(plan, bad, c)[:n]
    spoilt = torch.zeros((n, Hq), dtype=torch.bool, device="cuda")
    spoilt[1, 0] = spoilt[n - 1, Hq - 1] = True
    assert same(got[~spoilt], clean[~spoilt]) and got[spoilt].isnan().all()


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", FORMS)
def test_scales_from_flat_to_one_hot(scale, dtype, cache, D, Hq, Hkv):
    # where scores differ by thousands the largest takes all; the bound's share of the scores' fp32 sums grows with them
    for new, ctx in STEPS:
        plan = Plan(new, ctx, 32)
        c = new_cache(plan, Hkv, D, cache)
        q = randn(plan.rows, Hq, D, dtype=dtype)
        check(plan, attend(plan, q, c, scale), q, c, scale)


@pytest.mark.parametrize("cache", [F16, I8])
def test_a_captured_chunk_follows_the_plan_in_memory(cache):
    D, P, H = 64, 32, 3
    final = Plan([120, 60, 90], [500, 60, 2000], P, pad_rows=30)
    c = new_cache(final, H, D, cache)
    q = randn(final.rows, H, D)
    start, lens, out = final.q_start.clone(), final.ctx_len.clone(), torch.empty_like(q)

    def step():
        K.paged_attention(q, c[0], c[1], start, lens, final.table, None, c[2], c[3], out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for new, ctx in (([120, 60, 90], [500, 60, 2000]), ([1, 0, 200], [400, 60, 1900]), ([0, 0, 0], [0, 0, 0]), ([300, 0, 0], [512, 0, 0]), ([10, 10, 10], [0, 5, 2000])):
        plan = Plan(new, ctx, P)
        plan.table, plan.table_list, plan.width, plan.pages = final.table, final.table_list, final.width, final.pages
        start.copy_(plan.q_start)
        lens.copy_(plan.ctx_len)
        out.fill_(7)
        graph.replay()
        check(plan, out, q, c)
        assert (out[plan.starts[-1]:] == 7).all()


def test_calls_from_several_threads():
    import threading
    work = []
    for seed, (new, ctx, form) in enumerate([([1] * 9, [300] * 9, FORMS[0]), ([90, 40], [400, 90], FORMS[1]), ([200], [900], FORMS[2]), ([3, 2], [2000, 5], FORMS[3])]):
        dtype, cache, D, Hq, Hkv = form
        plan = Plan(new, ctx, 32, seed=seed)
        c = new_cache(plan, Hkv, D, cache)
        q = randn(plan.rows, Hq, D, dtype=dtype)
        work.append((plan, q, c, attend(plan, q, c), torch.cuda.Stream()))
    torch.cuda.synchronize()
    wrong = []

    def run(plan, q, c, want, stream):
        with torch.cuda.stream(stream):
            outs = [attend(plan, q, c) for _ in range(30)]
        stream.synchronize()
        wrong.extend(not same(o, want) for o in outs)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(wrong) == 120 and not any(wrong)
    for plan, q, c, want, _ in work:
        check(plan, want, q, c)
