"""The attention over the paged cache where numbers and plans go to extremes, against the plain form in 64 bits."""
import pytest
import torch

from generation import Plan, attention_64, attention_bound, new_cache
from pequegrad_b200 import kernels as K
from test_generation_gpu import attend, check, randn, same

pytestmark = pytest.mark.gpu

F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8

# new tokens, contexts, heads: tiles of sixteen rows; chunks whose keys are split over a cluster; chunks that are not split
SIZES = [([2, 3], [400, 700], 2), ([200], [700], 2), ([40] * 24, [520] * 24, 8), ([60] * 24, [520] * 24, 8)]


def check_numbers(plan, q, cache, got):
    """What is a number in the plain form is one, within the bound; the rest is NaN in both."""
    D = q.shape[-1]
    want, mass, size = attention_64(plan, q, cache, D ** -0.5)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{int(got.isnan().sum())} NaN for {int(nan.sum())}"
    mass = mass.nan_to_num(0)
    bound = attention_bound(want, mass, size, q.dtype, D, max(plan.ctx), float(mass.max()) * 4 + 1)
    err = (got.double() - want).abs()
    assert bool((err <= bound)[~nan].all()), float((err - bound)[~nan].max())
    assert K.device_error() == 0


@pytest.mark.parametrize("dtype,cache,D", [(F16, F16, 64), (BF16, BF16, 128), (F16, I8, 64), (BF16, I8, 128)])
@pytest.mark.parametrize("new,ctx", [([20] * 50, [0] * 50), ([60] * 50, [0] * 50), ([300] * 20 + [20] * 30, [-5] * 50), ([100] * 24 + [20] * 60, [300] * 24 + [0] * 60), ([150] * 12 + [1] * 90, [260] * 12 + [0] * 90), ([150] * 12 + [50] * 90, [260] * 12 + [0] * 90)])
def test_hundreds_of_work_items_without_a_key(new, ctx, dtype, cache, D):
    # several in a row for every CTA, alone and behind items with keys; with a table and without one
    H = 12
    plan = Plan(new, ctx, 32, pad_rows=2)
    c = new_cache(plan, H, D, cache)
    q = randn(plan.rows, H, D, dtype=dtype)
    outs = []
    for table in [plan.table] + ([plan.table[:, :0]] if max(ctx) <= 0 else []):
        out = torch.full_like(q, 7)
        plan.table = table
        attend(plan, q, c, out=out)
        check(plan, out, q, c)
        for b, n in enumerate(ctx):
            if n <= 0:
                assert (out[plan.starts[b]:plan.starts[b + 1]] == 0).all()
        assert (out[-2:] == 7).all()
        outs.append(out)
    assert same(outs[0], attend(plan, q, c, out=torch.full_like(q, 7)))


@pytest.mark.parametrize("cache", [F16, I8])
def test_waits_for_items_end_with_the_others(cache):
    # a launch that loads nothing and whose first items have no keys: roles that wait for items give up when nothing moves
    plan = Plan([60] * 60 + [200] * 4, [0] * 60 + [200] * 4, 32)
    c = new_cache(plan, 12, 64, cache)
    q = randn(plan.rows, 12, 64)
    K.gemm_wait_drill(1 << 14, skip_loads=True)
    attend(plan, q, c)
    torch.cuda.synchronize()
    code = K.device_error(reset=True)
    assert 32 <= code >> 16 <= 47
    check(plan, attend(plan, q, c), q, c)


@pytest.mark.parametrize("dtype,cache,D", [(F16, F16, 64), (BF16, BF16, 128), (F16, I8, 64)])
@pytest.mark.parametrize("new,ctx,H", [([200], [6000], 60), ([300] * 10, [400] * 10, 40)])
def test_waits_cut_short_leave_nothing_behind(new, ctx, H, dtype, cache, D):
    """Waits of so few polls run out in the middle of the work, or do not, in clusters with several rounds to go and outside. A
    launch that gave up says so, and the next one is right."""
    plan = Plan(new, ctx, 64)
    c = new_cache(plan, H, D, cache)
    q = randn(plan.rows, H, D, dtype=dtype)
    for polls in (1, 2, 8):
        K.gemm_wait_drill(polls, skip_loads=False)
        out = attend(plan, q, c)
        torch.cuda.synchronize()
        code = K.device_error(reset=True)
        assert code == 0 or 32 <= code >> 16 <= 47
        right = attend(plan, q, c)
        if polls == 1:
            check(plan, right, q, c)
            first = right
        assert same(right, first) and (code != 0 or same(out, first))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,ctx,H", SIZES)
@pytest.mark.parametrize("zeros", [128, 300])
def test_values_of_scale_zero_have_their_share_of_the_softmax(dtype, D, new, ctx, H, zeros):
    # whole blocks of keys whose values are zeros, stored with a scale of zero, before ordinary ones
    plan = Plan(new, ctx, 32)
    c = new_cache(plan, H, D, I8)
    for b in range(len(new)):
        for page, slot in plan.places(b, range(zeros)):
            c[3][page, :, slot] = 0
    q = randn(plan.rows, H, D, dtype=dtype)
    check(plan, attend(plan, q, c), q, c)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,ctx,H", SIZES)
def test_an_infinite_key(dtype, D, new, ctx, H):
    """Every second row has a score of +infinity, and with it no softmax; for the others that score is -infinity and the key
    does not count. At each place in eight neighbours, in a block that all rows see and in one that only some do."""
    plan = Plan(new, ctx, 32)
    q = randn(plan.rows, H, D, dtype=dtype)
    q[::2, 0, 3], q[1::2, 0, 3] = 1, -1
    clean = new_cache(plan, H, D, dtype)
    for at in [*range(136, 144), *range(ctx[0] - 8, ctx[0])]:
        c = (clean[0].clone(), *clean[1:])
        page, slot = plan.places(0, [at])[0]
        c[0][page, 0, slot, 3] = float("inf")
        check_numbers(plan, q, c, attend(plan, q, c))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,ctx,H", SIZES + [([1], [1], 2), ([150], [150], 2)])
def test_rows_whose_every_score_is_minus_infinity(dtype, D, new, ctx, H):
    """They have keys, so they are not rows without one: minus infinity less itself is NaN in the plain softmax. Head 1 is
    left alone; in head 0 all keys are infinite, or those of the first 200 positions, which then do not count."""
    plan = Plan(new, ctx, 32)
    q = randn(plan.rows, H, D, dtype=dtype)
    q[:, 0, 3] = -1
    for first in (max(ctx), 200):
        c = new_cache(plan, H, D, dtype)
        for b, n in enumerate(ctx):
            for page, slot in plan.places(b, range(min(first, n))):
                c[0][page, 0, slot, 3] = float("inf")
        check_numbers(plan, q, c, attend(plan, q, c))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,ctx,H", SIZES)
@pytest.mark.parametrize("where", ["early", "last"])
def test_value_scales_of_any_ratio(dtype, D, new, ctx, H, where):
    """One token's values are 2^26 times the others', and nobody looks at it: it lies 60 below the other scores, or it is the
    last token, which only one row sees. What the others give must not be rounded away beside it.

    Probabilities times value scales are rounded to fp16 relative to the row's largest such product, P >= 1 of its scale: what
    is below 2^-25 of it is dropped. The key that has it also has a value of at least 64 of the 127 among its 64 or more, so
    each key loses at most 2^-25 * 127 <= 2^-24 of the row's largest sum of |p v|."""
    plan = Plan(new, ctx, 32)
    c = new_cache(plan, H, D, I8)
    c[3].mul_(2.0 ** -12)
    q = randn(plan.rows, H, D, dtype=dtype).abs() + 0.5
    for b, n in enumerate(ctx):
        page, slot = plan.places(b, [150 if where == "early" else n - 1])[0]
        c[3][page, :, slot] = 2.0 ** 8
        if where == "early":
            c[0][page, :, slot], c[2][page, :, slot] = -127, 0.1
    got = attend(plan, q, c)
    want, mass, size = attention_64(plan, q, c, D ** -0.5)
    bound = attention_bound(want, mass, size, dtype, D, 0, 0.0) + max(ctx) * 2.0 ** -24 * mass.amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float((err / mass).max()))
    assert K.device_error() == 0


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", [(F16, F16, 64, 4, 4), (BF16, BF16, 128, 8, 2), (F16, I8, 128, 6, 2), (BF16, I8, 64, 20, 1)])
@pytest.mark.parametrize("new,ctx", [([1, 3, 0, 2], [700, 40, 9, 2000]), ([200, 1, 64], [700, 5, 90]), ([90] * 30, [300] * 30)])
def test_the_result_may_take_the_queries_place(new, ctx, dtype, cache, D, Hq, Hkv):
    plan = Plan(new, ctx, 32, pad_rows=2)
    c = new_cache(plan, Hkv, D, cache)
    qkv = randn(plan.rows, Hq + 2 * Hkv, D, dtype=dtype)
    keep = qkv.clone()
    want = attend(plan, keep[:, :Hq], c, out=keep[:, :Hq].clone())
    assert attend(plan, qkv[:, :Hq], c, out=qkv[:, :Hq]) is not None
    assert same(qkv[:, :Hq], want) and same(qkv[:, Hq:], keep[:, Hq:])


def test_results_that_share_memory_are_refused():
    H, D, P = 2, 64, 16
    plan = Plan([5, 3], [20, 9], P)
    n = plan.kv_starts[-1]
    kc, vc, _, _ = new_cache(plan, H, D, F16)
    k8, v8, ks, vs = new_cache(plan, H, D, I8)
    at = (plan.q_start, plan.ctx_len, plan.table)
    buf = randn(n + 1, 3, H, D)
    keep = [x.clone() for x in (kc, vc, buf, ks, vs)]

    def refused(call, *names):
        with pytest.raises(Exception, match="shares memory") as e:
            call()
        assert all(name in str(e.value) for name in names), str(e.value)

    x = buf[:plan.rows]
    refused(lambda: K.kv_write(x[:, 0], x[:, 1], kc, kc, *at), "v_cache", "k_cache")
    refused(lambda: K.kv_write(x[:, 0], x[:, 1], kc[1:], kc[:-1], *at), "v_cache", "k_cache")
    refused(lambda: K.kv_write(x[:, 0], x[:, 1], k8, v8, *at, ks, ks), "k_scale", "v_scale")
    refused(lambda: K.kv_write(kc.view(-1, H, D)[3:3 + plan.rows], x[:, 1], kc, vc, *at), "k_cache")
    refused(lambda: K.kv_read(kc, vc, plan.kv_start, plan.table, n, out=(buf[:n, 0], buf[:n, 0])), "k", "v")
    refused(lambda: K.kv_read(kc, vc, plan.kv_start, plan.table, n, out=(buf[:n, 0], buf[1:, 0])), "k", "v")
    refused(lambda: K.kv_read(kc, vc, plan.kv_start, plan.table, 2, out=(buf[:2, 0], vc.view(-1, H, D)[:2])), "v_cache")
    refused(lambda: K.paged_attention(x[:, 0], kc, vc, *at, out=x.flatten(1, 2)[:, 1:1 + H]), "out", "q")
    refused(lambda: K.paged_attention(buf[:plan.rows, 0], kc, vc, *at, out=buf[1:plan.rows + 1, 0]), "out", "q")
    refused(lambda: K.paged_attention(x[:, 0], kc, vc, *at, out=vc.view(-1, H, D)[:plan.rows]), "v_cache")
    rows = torch.randn((4, 40), device="cuda")
    refused(lambda: K.logits_process(rows[:, :30], out=rows[:, 1:31]))
    refused(lambda: K.logits_process(rows[:3], out=rows[1:]))
    refused(lambda: K.logits_process(rows, bias_ids=torch.zeros((4, 2), dtype=torch.int32, device="cuda"), bias=rows[:, :2], out=rows))
    for a, b in zip((kc, vc, buf, ks, vs), keep):
        assert same(a, b)
    # neighbours in one buffer are apart
    K.kv_read(kc, vc, plan.kv_start, plan.table, n, out=(buf[:n, 0], buf[:n, 2]))
    both = torch.zeros((plan.pages, 2, H, P, D), dtype=F16, device="cuda")
    K.kv_write(x[:, 0], x[:, 1], both[:, 0], both[:, 1], *at)
    K.paged_attention(x[:, 0], kc, vc, *at, out=x[:, 1])
    K.logits_process(rows[:, :20], out=rows[:, 20:])
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", [(F16, F16, 64, 12, 12), (BF16, BF16, 128, 16, 16), (F16, I8, 128, 6, 2), (BF16, I8, 64, 15, 5), (F16, F16, 128, 18, 1)])
@pytest.mark.parametrize("new,ctx", [([5] * 4, [3000] * 4), ([2, 4, 1, 3], [2500, 31, 700, 4000]), ([5, 5], [129, 128])])
def test_a_few_tokens_over_long_contexts(new, ctx, dtype, cache, D, Hq, Hkv):
    # rows that begin no tile beside clusters whose keys are split as far as they go
    plan = Plan(new, ctx, 64, pad_rows=3)
    c = new_cache(plan, Hkv, D, cache)
    q = randn(plan.rows, Hq, D, dtype=dtype)
    out = torch.full_like(q, 7)
    attend(plan, q, c, out=out)
    check(plan, out, q, c)
    assert (out[plan.starts[-1]:] == 7).all() and same(out[:plan.starts[-1]], attend(plan, q, c)[:plan.starts[-1]])


@pytest.mark.parametrize("dtype,cache,D,Hq,Hkv", [(F16, F16, 64, 2, 2), (BF16, BF16, 128, 6, 2), (F16, I8, 64, 5, 1), (BF16, I8, 128, 16, 2), (F16, F16, 64, 15, 1)])
def test_every_row_of_uneven_sequences_is_found(dtype, cache, D, Hq, Hkv):
    """Numbers of new tokens around those of a tile, in every order, empty sequences between them, offsets that do not begin at
    zero: the rows kernel deals its tiles out by slots of which some are empty, and every tile must have one."""
    g = torch.Generator().manual_seed(5)
    for case in range(12):
        n = int(torch.randint(1, 40, (), generator=g))
        new = torch.randint(0, (2, 4, 18, 34)[case % 4], (n,), generator=g).tolist()
        limit = 16 * n * Hkv // Hq  # on average, for the rows kernel
        while sum(new) > limit:
            new[new.index(max(new))] //= 2
        ctx = [x + int(torch.randint(0, 90, (), generator=g)) for x in new]
        plan = Plan(new, ctx, 16, seed=case, pad_rows=3)
        c = new_cache(plan, Hkv, D, cache)
        q = randn(plan.rows, Hq, D, dtype=dtype, seed=case)
        for skip in (0, 5):
            plan.q_start = torch.tensor([s + skip for s in plan.starts], dtype=torch.int32, device="cuda")
            out = torch.full((plan.rows + skip, Hq, D), 7.0, dtype=dtype, device="cuda")
            attend(plan, torch.cat([q[:skip], q]), c, out=out)
            check(plan, out[skip:], q, c)
            assert (out[:skip] == 7).all() and (out[plan.starts[-1] + skip:] == 7).all()


@pytest.mark.parametrize("new,nats", [(1, 14.5), (1, 18.0), (3, 18.0), (40, 14.5), (60, 14.5)])
@pytest.mark.parametrize("dtype,cache,D", [(F16, F16, 64), (F16, I8, 64), (BF16, I8, 128), (F16, F16, 128)])
def test_many_small_probabilities_beside_one_that_is_not(new, nats, dtype, cache, D):
    """One key lies 14.5 or 18 above 60000 others: each has a probability of 2^-21 or 2^-26, and together they make 3 % or 0.1 %
    of the row. Probabilities are rounded to 16 bits, relative to their size as long as they are normal numbers there; nothing
    is allowed for those that are not."""
    H, n = 2, 60000
    plan = Plan([new], [n], 64)
    c = new_cache(plan, H, D, cache)
    k = torch.zeros((n, H, D), dtype=dtype, device="cuda")
    k[0] = nats / D ** 0.5
    v = randn(n, H, D, dtype=dtype, seed=1).abs() + 0.5
    v[0] = 0
    full = Plan([n], [n], 64)
    K.kv_write(k, v, c[0], c[1], full.q_start, full.ctx_len, plan.table, c[2], c[3])
    q = torch.ones((new, H, D), dtype=dtype, device="cuda")
    got = attend(plan, q, c)
    want, mass, size = attention_64(plan, q, c, D ** -0.5)
    err = (got.double() - want).abs()
    bound = attention_bound(want, mass, size, dtype, D, 0, 0.0)
    assert bool((err <= bound).all()), (float((err / want).max()), float((bound / want).max()))
