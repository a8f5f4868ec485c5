"""The paged cache, the attention over it and the logit shaping, against plain forms in 64 bits."""
import pytest
import torch

from generation import Plan, attention_64, attention_bound, gather, logits_64, new_cache, quantised
from pequegrad_b200 import kernels as K

pytestmark = pytest.mark.gpu

F16, BF16, F32, I8 = torch.float16, torch.bfloat16, torch.float32, torch.int8


def bits(x):
    return x.contiguous().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def same(a, b):
    return torch.equal(bits(a), bits(b))


def randn(*shape, dtype=F16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


# ---- the cache -------------------------------------------------------------------------------------------------------

PLANS = [([1, 1, 1], [5, 16, 33]), ([3, 0, 17, 40], [3, 9, 70, 40]), ([0], [0]), ([], []), ([130], [300]), ([1] * 70, list(range(1, 71)))]


@pytest.mark.parametrize("new,ctx", PLANS)
@pytest.mark.parametrize("dtype,D,P,H,layout", [(F16, 64, 16, 3, "hpd"), (BF16, 128, 64, 2, "phd"), (F16, 128, 128, 5, "hpd"), (BF16, 64, 32, 1, "phd")])
def test_write_copies_the_rows_and_nothing_else(new, ctx, dtype, D, P, H, layout):
    plan = Plan(new, ctx, P, pad_rows=3)
    kc, vc, _, _ = new_cache(plan, H, D, dtype, layout)
    want_k, want_v = kc.clone(), vc.clone()
    # rows inside a packed projection, as a model has them
    qkv = randn(plan.rows, 3, H, D, dtype=dtype)
    k, v = qkv[:, 1], qkv[:, 2]
    for b, n in enumerate(plan.new):
        for i, (page, slot) in enumerate(plan.places(b, range(plan.ctx[b] - n, plan.ctx[b]))):
            want_k[page, :, slot] = k[plan.starts[b] + i]
            want_v[page, :, slot] = v[plan.starts[b] + i]
    K.kv_write(k, v, kc, vc, plan.q_start, plan.ctx_len, plan.table)
    assert same(kc, want_k) and same(vc, want_v)


@pytest.mark.parametrize("new,ctx", PLANS)
@pytest.mark.parametrize("dtype,D,P,H,layout", [(F16, 64, 16, 3, "hpd"), (BF16, 128, 64, 2, "phd"), (F16, 128, 32, 1, "phd"), (BF16, 64, 128, 4, "hpd")])
def test_write_quantises_each_token_and_head(new, ctx, dtype, D, P, H, layout):
    plan = Plan(new, ctx, P, pad_rows=2)
    kc, vc, ks, vs = new_cache(plan, H, D, I8, layout)
    k, v = randn(plan.rows, H, D, dtype=dtype, seed=1) * 4, randn(plan.rows, H, D, dtype=dtype, seed=2)
    want = [c.clone() for c in (kc, vc, ks, vs)]
    for x, wq, ws in ((k, want[0], want[2]), (v, want[1], want[3])):
        q, s = quantised(x)
        for b, n in enumerate(plan.new):
            for i, (page, slot) in enumerate(plan.places(b, range(plan.ctx[b] - n, plan.ctx[b]))):
                wq[page, :, slot] = q[plan.starts[b] + i].cuda()
                ws[page, :, slot] = s[plan.starts[b] + i].cuda()
    K.kv_write(k, v, kc, vc, plan.q_start, plan.ctx_len, plan.table, k_scale=ks, v_scale=vs)
    for got, w in zip((kc, vc, ks, vs), want):
        assert same(got, w)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantised_values_at_the_edges(dtype):
    D, P = 64, 16
    fin = torch.finfo(dtype)
    rows = [torch.zeros(D), torch.full((D,), 1e-8), torch.full((D,), float(fin.tiny)), torch.full((D,), float(fin.max)),
            torch.arange(D) - 31.5,                                          # 31.5 / s and its neighbours
            torch.cat([torch.tensor([127.0]), torch.arange(1, D) - 32 + 0.5]),  # s = 1: every value but one is a tie
            torch.cat([torch.tensor([-127.0]), torch.arange(1, D) - 32 + 0.5]),
            torch.cat([torch.tensor([float("nan")]), torch.ones(D - 1)]), torch.cat([torch.ones(D - 1), torch.tensor([float("-inf")])]),
            torch.full((D,), -0.0)]
    x = torch.stack(rows).to(dtype).cuda()[:, None]
    n = len(rows)
    plan = Plan([n], [n], P)
    kc, vc, ks, vs = new_cache(plan, 1, D, I8)
    K.kv_write(x, -x, kc, vc, plan.q_start, plan.ctx_len, plan.table, k_scale=ks, v_scale=vs)
    back = K.kv_read(kc, vc, plan.kv_start, plan.table, n, ks, vs, out_dtype=F32)
    for got, src in zip(back, (x, -x)):
        q, s = quantised(src)
        want = q.float() * s[..., None]
        assert torch.equal(got.cpu().isnan(), want.isnan()) and torch.equal(got.cpu().nan_to_num(), want.nan_to_num())
    assert back[0][7].isnan().all() and back[0][8].isnan().all()  # nothing made up for a head that has no int8 form


@pytest.mark.parametrize("ctx", [[5, 16, 0, 33], [1], [0, 0], [], [700, 3, 129]])
@pytest.mark.parametrize("cache,out,D,P,H,layout", [(F16, F16, 64, 16, 3, "hpd"), (BF16, BF16, 128, 32, 2, "phd"), (I8, F16, 64, 64, 2, "phd"),
                                                    (I8, BF16, 128, 128, 3, "hpd"), (I8, F32, 64, 16, 1, "hpd"), (I8, F32, 128, 32, 2, "phd")])
def test_read_gathers_and_dequantises(ctx, cache, out, D, P, H, layout):
    plan = Plan([0] * len(ctx), ctx, P)
    kc, vc, ks, vs = new_cache(plan, H, D, cache, layout)
    n = plan.kv_starts[-1]
    # two rows behind the last sequence keep what they hold; the outputs are the halves of one buffer
    buf = torch.full((n + 2, 2, H, D), 7.0, dtype=out, device="cuda")
    k, v = K.kv_read(kc, vc, plan.kv_start, plan.table, n + 2, ks, vs, out=(buf[:, 0], buf[:, 1]))
    for got, c, s in ((k, kc, ks), (v, vc, vs)):
        want = [torch.full((0, H, D), 0.0, device="cuda").to(out)]
        for b in range(len(ctx)):
            x, _ = gather(plan, b, ctx[b], c, None)
            if s is not None:
                x = x.float() * gather(plan, b, ctx[b], s[..., None], None)[0].float()
            want.append(x.to(out))
        assert same(got[:n], torch.cat(want))
    assert (buf[n:] == 7).all()


def test_positions_without_a_page():
    D, P, H = 64, 16, 2
    plan = Plan([40, 20, 3], [40, 20, 3], P, spare_pages=4, spare_width=0)
    # an entry that is no page (two kinds), a table that is too short for a sequence
    plan.table_list[0][1], plan.table_list[1][0], plan.table_list[2][0] = -1, plan.pages, 2 ** 31 - 1
    plan.table = torch.tensor(plan.table_list, dtype=torch.int32, device="cuda")[:, :2].contiguous()
    plan.table_list, plan.width = [t[:2] for t in plan.table_list], 2
    for dtype in (F16, I8):
        cache = new_cache(plan, H, D, dtype)
        before = [c.clone() for c in cache if c is not None]
        x = randn(plan.rows, H, D)
        K.kv_write(x, x, cache[0], cache[1], plan.q_start, plan.ctx_len, plan.table, cache[2], cache[3])
        for c, old in zip([c for c in cache if c is not None], before):
            there = torch.zeros(c.shape[0], P, dtype=torch.bool)
            for b, n in enumerate(plan.ctx):
                for page, slot in plan.places(b, range(n)):
                    if page is not None:
                        there[page, slot] = True
            kept = ~there[:, None].expand(c.shape[:3])
            assert same(c[kept.cuda()], old[kept.cuda()])
        k, _ = K.kv_read(cache[0], cache[1], plan.kv_start, plan.table, plan.rows, cache[2], cache[3], out_dtype=F16)
        for b, n in enumerate(plan.ctx):
            for i, (page, _) in enumerate(plan.places(b, range(n))):
                got = k[plan.kv_starts[b] + i]
                assert (got == 0).all() if page is None else (dtype == I8 or same(got, x[plan.starts[b] + i]))
    # contexts shorter than their new rows: the first rows stand before position zero
    plan = Plan([10, 4], [4, 0], P)
    kc, vc, _, _ = new_cache(plan, H, D, F16, fill=0)
    x = randn(plan.rows, H, D)
    K.kv_write(x, x, kc, vc, plan.q_start, plan.ctx_len, plan.table)
    k, _ = K.kv_read(kc, vc, plan.kv_start, plan.table, 4)
    assert same(k, x[6:10]) and int((kc != 0).any(-1).any(1).sum()) == 4


# ---- attention -------------------------------------------------------------------------------------------------------

def attend(plan, q, cache, scale=None, out=None):
    return K.paged_attention(q, cache[0], cache[1], plan.q_start, plan.ctx_len, plan.table, scale, cache[2], cache[3], out=out)


def check(plan, got, q, cache, scale=None):
    D = q.shape[-1]
    want, mass, size = attention_64(plan, q, cache, D ** -0.5 if scale is None else scale)
    n = plan.starts[-1]
    vmax = float(mass.max()) * 4 + 1 if mass.numel() else 1.0
    bound = attention_bound(want, mass, size, q.dtype, D, max(0, max(plan.ctx, default=0)), vmax)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)[:n]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err - bound)[:n].max()):.3g} at {bad.nonzero()[0].tolist()}"
    assert K.device_error() == 0


ATTENTION = [
    # new, ctx                                              one token: nothing but itself, a page, a page and one, far
    ([1], [1]), ([1], [16]), ([1], [17]), ([1] * 5, [1, 31, 128, 700, 64]), ([1, 0, 1, 0], [9, 33, 260, 0]),
    # a few tokens
    ([2, 3, 1], [2, 300, 5]), ([4], [1000]), ([7, 5], [7, 260]),
    # chunks: short of a tile, a tile, more; with and without context; ragged, mixed with single tokens
    ([40], [40]), ([100, 30], [100, 200]), ([128], [128]), ([129], [400]), ([300, 1, 0, 64], [300, 500, 20, 191]), ([257], [1025]),
]
FORMS = [(F16, F16, 64, 16, 2, 2, "hpd"), (BF16, BF16, 128, 32, 4, 2, "phd"), (F16, I8, 64, 64, 3, 3, "hpd"), (BF16, I8, 128, 128, 8, 1, "phd"),
         (BF16, I8, 64, 16, 6, 2, "phd"), (F16, F16, 128, 64, 5, 1, "hpd"), (F16, I8, 128, 32, 16, 2, "hpd"), (BF16, BF16, 64, 128, 7, 1, "phd")]


@pytest.mark.parametrize("dtype,cache,D,P,Hq,Hkv,layout", FORMS)
@pytest.mark.parametrize("new,ctx", ATTENTION)
def test_attention(new, ctx, dtype, cache, D, P, Hq, Hkv, layout):
    plan = Plan(new, ctx, P, pad_rows=2)
    c = new_cache(plan, Hkv, D, cache, layout)
    qkv = randn(plan.rows, Hq + 2 * Hkv, D, dtype=dtype, seed=3)
    out = torch.full((plan.rows, Hq, D), 7.0, dtype=dtype, device="cuda")
    attend(plan, qkv[:, :Hq], c, out=out)
    check(plan, out, qkv[:, :Hq], c)
    assert (out[plan.starts[-1]:] == 7).all()  # rows behind the last sequence


@pytest.mark.parametrize("dtype,cache,D,P,Hq,Hkv", [(F16, F16, 64, 16, 12, 12), (F16, I8, 64, 32, 12, 12), (BF16, I8, 128, 64, 20, 20), (BF16, BF16, 128, 128, 20, 20)])
@pytest.mark.parametrize("new,ctx", [([100, 90], [3000, 5000]), ([300, 64, 129], [4000, 4100, 2000]), ([90] * 20, [2000] * 20)])
def test_halves_of_a_tile_that_end_apart(new, ctx, dtype, cache, D, P, Hq, Hkv):
    # tiles whose second half is empty, short or a block longer, over many blocks of keys, several times in a row
    plan = Plan(new, ctx, P)
    c = new_cache(plan, Hkv, D, cache)
    q = randn(plan.rows, Hq, D, dtype=dtype)
    outs = [attend(plan, q, c) for _ in range(3)]
    check(plan, outs[0], q, c)
    assert same(outs[0], outs[1]) and same(outs[0], outs[2])


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_scores_that_grow_and_shrink(new, cache):
    # the running maximum moves in every block, upwards and downwards, by more than fp16 spans
    D, P, H = 64, 32, 2
    plan = Plan([new, new], [900, 900], P)
    c = new_cache(plan, H, D, cache)
    ramp = torch.linspace(-8, 8, 900, device="cuda")
    for b, sign in enumerate((1, -1)):
        k = (sign * ramp)[:, None, None].expand(900, H, D)
        one = Plan([900], [900], P)
        one.pages, one.table = plan.pages, plan.table[b:b + 1]
        K.kv_write(k.half().contiguous(), randn(900, H, D, seed=b), c[0], c[1], one.q_start, one.ctx_len, one.table, c[2], c[3])
    q = torch.ones((plan.rows, H, D), dtype=F16, device="cuda")
    q[::2] = -1
    for scale in (0.125, 1.0, 0.01):
        check(plan, attend(plan, q, c, scale), q, c, scale)


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_very_different_size(cache, D):
    # one token's values are 2^13 times the others', and it is hardly looked at: what the others give must not drown
    P, H = 16, 2
    for new in (1, 70):
        plan = Plan([new], [400], P)
        c = new_cache(plan, H, D, cache)
        k, v = randn(400, H, D, seed=5) * 0.1, randn(400, H, D, seed=6) * 0.01
        k[200], v[200] = -4.0, 80.0
        full = Plan([400], [400], P)
        K.kv_write(k, v, c[0], c[1], full.q_start, full.ctx_len, plan.table, c[2], c[3])
        q = randn(new, H, D, seed=7).abs() + 0.5
        check(plan, attend(plan, q, c), q, c)


@pytest.mark.parametrize("dtype,cache,D,P", [(F16, F16, 64, 16), (BF16, BF16, 128, 64), (F16, I8, 64, 32), (BF16, I8, 128, 128)])
@pytest.mark.parametrize("new,ctx", [([1, 1], [5, 130]), ([60, 3], [60, 190]), ([140], [140])])
def test_slots_behind_the_context_may_hold_anything(new, ctx, dtype, cache, D, P):
    plan = Plan(new, ctx, P, spare_pages=3)
    H = 2
    for junk in (float("nan"), float("inf"), float("-inf")):
        c = new_cache(plan, H, D, cache)
        used = torch.zeros(plan.pages, P, dtype=torch.bool)
        for b, n in enumerate(ctx):
            for page, slot in plan.places(b, range(n)):
                used[page, slot] = True
        free = (~used).cuda()[:, None].expand(plan.pages, H, P)
        for x in (c[:2] if cache != I8 else c[2:]):
            x[free] = junk
        q = randn(plan.rows, H, D, dtype=dtype)
        check(plan, attend(plan, q, c), q, c)


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [5, 130, 40]), ([60, 2, 40], [60, 190, 40]), ([140, 130, 10], [300, 130, 20])])
def test_keys_without_a_page_are_left_out(new, ctx, cache):
    # the first page of the first sequence is gone, one inside the second; the third has none at all: zeros
    D, P, H = 64, 32, 2
    plan = Plan(new, ctx, P)
    plan.table_list[0][0] = -1
    plan.table_list[1][2] = plan.pages + 5
    plan.table_list[2] = [-1] * plan.width
    plan.table = torch.tensor(plan.table_list, dtype=torch.int32, device="cuda")
    c = new_cache(plan, H, D, cache)
    q = randn(plan.rows, H, D)
    out = attend(plan, q, c)
    check(plan, out, q, c)
    assert (out[plan.starts[2]:] == 0).all()
    # a context that claims more than the table holds sees what the table holds; rows before position zero see nothing
    plan = Plan([2, 9, 150], [32, 5, 100], P, spare_width=0)
    q = randn(plan.rows, H, D)
    c = new_cache(plan, H, D, cache)
    plan.ctx_len = torch.tensor([32, 5, 100], dtype=torch.int32, device="cuda")
    out = attend(plan, q, c)
    check(plan, out, q, c)
    assert (out[2:6] == 0).all() and (out[11:61] == 0).all()
    plan.ctx[0] = plan.width * P + 1000
    plan.ctx_len[0] = plan.ctx[0]
    plan.table_list[0] = plan.table_list[2]
    plan.table[0] = plan.table[2]
    check(plan, attend(plan, q, c), q, c)


@pytest.mark.parametrize("dtype,cache,D,P", [(F16, F16, 64, 16), (BF16, BF16, 128, 64), (BF16, BF16, 64, 32), (F16, F16, 128, 16), (F16, I8, 64, 32), (BF16, I8, 128, 128)])
@pytest.mark.parametrize("new,ctx", [(3, 40), (16, 16), (9, 137), (200, 200), (260, 700), (130, 3000)])
def test_a_token_that_is_not_a_number_reaches_only_the_rows_that_see_it(new, ctx, dtype, cache, D, P):
    """NaN and infinities in the values (int8: in the scales) and in the keys of new tokens. The rows before such a token give
    what they would without it; of the rows that see it, a bad value spoils its column, a bad key or scale the row."""
    H, plan = 2, Plan([new], [ctx], P)
    k, v = randn(ctx, H, D, dtype=dtype, seed=1), randn(ctx, H, D, dtype=dtype, seed=2)
    q = randn(new, H, D, dtype=dtype, seed=3)
    full = Plan([ctx], [ctx], P)
    first = ctx - new
    for where in sorted({new - 1, new // 2, 1}):
        at = first + where
        for what in ("v nan", "v inf", "v both", "k nan"):
            c = new_cache(plan, H, D, cache)
            K.kv_write(k, v, c[0], c[1], full.q_start, full.ctx_len, plan.table, c[2], c[3])
            want, mass, size = attention_64(plan, q, c, D ** -0.5)
            bad = v.clone() if what[0] == "v" else k.clone()
            if what == "v nan":
                bad[at, 0, 5] = float("nan")
            elif what == "v inf":
                bad[at, 1, D - 1], bad[at, 0, 0] = float("-inf"), float("inf")
            elif what == "v both":
                bad[at, 0, 7], bad[at - 1, 0, 7] = float("inf"), float("-inf")
            else:
                bad[at, 1, 3] = float("nan")
            K.kv_write(bad if what[0] == "k" else k, bad if what[0] == "v" else v, c[0], c[1], full.q_start, full.ctx_len, plan.table, c[2], c[3])
            got = attend(plan, q, c)
            clean = torch.ones((new, H, D), dtype=torch.bool, device="cuda")
            if cache == I8:  # a head with such a value has no int8 form: all of it reads as NaN
                heads = {"v nan": [0], "v inf": [0, 1], "v both": [0], "k nan": [1]}[what]
                clean[max(0, where - (what == "v both")):, heads] = False
                expect = torch.full_like(want, float("nan"))
            else:
                expect = torch.zeros_like(want)
                if what == "k nan":
                    expect[where:, 1] = float("nan")
                    clean[where:, 1] = False
                else:
                    for j in (at - 1, at):
                        b = bad[j].double()
                        spoilt = ~torch.isfinite(b)
                        rows = slice(max(0, j - first), None)
                        expect[rows] += torch.where(spoilt, b, torch.zeros_like(b))
                        clean[rows] &= ~spoilt
            bound = attention_bound(want, mass, size, dtype, D, ctx, float(mass.max()) * 4 + 1)
            err = (got.double() - want).abs()
            assert bool((err <= bound)[clean].all()), (what, where)
            g, e = got.double()[~clean], expect[~clean]
            assert torch.equal(g.isnan(), e.isnan()) and torch.equal(g[~e.isnan()], e[~e.isnan()]), (what, where)


@pytest.mark.parametrize("new,ctx", [([1, 2], [100, 40]), ([130], [130]), ([20, 0, 70], [500, 3, 70])])
@pytest.mark.parametrize("Hq,Hkv,cache,D", [(20, 1, F16, 64), (48, 2, I8, 128), (64, 1, BF16, 128), (17, 1, I8, 64)])
def test_many_query_heads_share_a_key_head(new, ctx, Hq, Hkv, cache, D):
    # more than sixteen heads of one token, and numbers that divide no tile
    dtype = BF16 if cache == BF16 else F16
    plan = Plan(new, ctx, 32, pad_rows=1)
    c = new_cache(plan, Hkv, D, cache)
    q = randn(plan.rows, Hq, D, dtype=dtype)
    check(plan, attend(plan, q, c), q, c)


def test_two_streams_at_once_and_nothing_at_all():
    plans = [Plan([1] * 30, [300 + 10 * i for i in range(30)], 16, seed=1), Plan([200, 90], [700, 800], 64, seed=2)]
    work = []
    for plan, (Hq, Hkv, D, cache) in zip(plans, ((12, 12, 64, F16), (8, 2, 128, I8))):
        c = new_cache(plan, Hkv, D, cache)
        q = randn(plan.rows, Hq, D)
        work.append((plan, q, c, attend(plan, q, c)))
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, (plan, q, c, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attend(plan, q, c))
    torch.cuda.synchronize()
    for i, (plan, q, c, alone) in enumerate(work):
        check(plan, alone, q, c)
        assert all(same(o, alone) for o in outs[i])
    # no rows; no sequences; sequences without rows; a cache without pages
    for new, ctx, pad in (([], [], 0), ([], [], 3), ([0, 0], [5, 0], 2)):
        plan = Plan(new, ctx, 16, pad_rows=pad)
        c = new_cache(plan, 2, 64, F16)
        q = randn(plan.rows, 2, 64)
        out = torch.full_like(q, 7)
        attend(plan, q, c, out=out)
        assert (out == 7).all()
    plan = Plan([3, 200], [3, 200], 16)
    c = tuple(torch.empty((0, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2)) + (None, None)
    assert (attend(plan, randn(203, 2, 64), c) == 0).all()
    K.kv_write(randn(203, 2, 64), randn(203, 2, 64), c[0], c[1], plan.q_start, plan.ctx_len, plan.table)
    assert (K.kv_read(c[0], c[1], plan.kv_start, plan.table, 203)[0] == 0).all()


@pytest.mark.parametrize("cache", [F16, I8])
def test_a_wait_that_runs_out_is_reported(cache):
    """The next chunk launch loads nothing and its waits give up early: it records who gave up and returns, in clusters too;
    launches do nothing until the word is cleared, and then the same call is right again."""
    for new, ctx, H in (([200], [2000], 2), ([300] * 6, [300] * 6, 40)):
        plan = Plan(new, ctx, 32)
        c = new_cache(plan, H, 64, cache)
        q = randn(plan.rows, H, 64)
        check(plan, attend(plan, q, c), q, c)
        K.gemm_wait_drill(1024, skip_loads=True)
        out = torch.full_like(q, 7)
        attend(plan, q, c, out=out)
        torch.cuda.synchronize()
        again = torch.full_like(q, 7)
        attend(plan, q, c, out=again)
        torch.cuda.synchronize()
        code = K.device_error(reset=True)
        assert 32 <= code >> 16 <= 47 and (out == 7).all() and (again == 7).all()
        check(plan, attend(plan, q, c), q, c)


def test_many_sequences_and_heads():
    # more work than the GPU holds at once, of very different lengths
    for new, P, form in ([1] * 200, 16, (F16, F16, 64, 12, 12)), ([1, 90, 2, 0, 33, 1, 128] * 12, 64, (BF16, BF16, 128, 8, 2)), ([5, 1, 20] * 40, 32, (F16, I8, 64, 12, 4)):
        dtype, cache, D, Hq, Hkv = form
        ctx = [n + (37 * i * i) % 500 for i, n in enumerate(new)]
        plan = Plan(new, ctx, P)
        c = new_cache(plan, Hkv, D, cache)
        q = randn(plan.rows, Hq, D, dtype=dtype)
        out = attend(plan, q, c)
        check(plan, out, q, c)
        assert same(out, attend(plan, q, c))  # the same bits again


def test_a_long_context_and_pages_past_four_gigabytes():
    # 70000 cached tokens of one sequence, in pages whose offsets pass 2^32 bytes
    D, P, H, n = 64, 128, 2, 70000
    pages = (1 << 32) // (H * P * D * 2) + 1000
    kc, vc = (torch.empty((pages, H, P, D), dtype=F16, device="cuda") for _ in range(2))
    plan = Plan([1], [n], P)
    need = -(-n // P)
    g = torch.Generator().manual_seed(2)
    order = (torch.randperm(need, generator=g) + pages - need).tolist()
    plan.table_list, plan.pages = [order + [-1]], pages
    plan.table = torch.tensor(plan.table_list, dtype=torch.int32, device="cuda")
    x = randn(n, 2, H, D, seed=4)
    full = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    K.kv_write(x[:, 0], x[:, 1], kc, vc, full, plan.ctx_len, plan.table)
    k, v = K.kv_read(kc, vc, full, plan.table, n)
    assert same(k, x[:, 0]) and same(v, x[:, 1])
    for new in (1, 200):
        p = Plan([new], [n], P)
        p.table_list, p.pages, p.table = plan.table_list, pages, plan.table
        q = randn(new, H, D)
        check(p, attend(p, q, (kc, vc, None, None)), q, (kc, vc, None, None))


def test_contexts_shorter_than_their_new_rows():
    # more sequences than a warp looks at together, none of which has a key for any row; then some that have
    for ctx in ([0] * 45, [-3] * 40, [0] * 33 + [25] * 20):
        for new in (1, 20, 300):
            plan = Plan([new] * len(ctx), ctx, 16, pad_rows=1)
            c = new_cache(plan, 2, 64, F16)
            q = randn(plan.rows, 2, 64)
            out = torch.full_like(q, 7)
            attend(plan, q, c, out=out)
            check(plan, out, q, c)
            assert (out[: new * ctx.count(ctx[0])] == 0).all() and (out[-1] == 7).all()


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("new", [1, 32])
def test_a_context_of_millions_of_tokens(new, cache):
    """A table that names one page over and over: key j of the page counts as often as it is seen. A role may wait for as long
    as an item takes, which here is tens of milliseconds, and the second item of a CTA as long again."""
    D, P, H = 64, 128, 160
    ctx = (1 << 22) + 37
    plan = Plan([new], [ctx], P, spare_pages=0)
    plan.pages = 1
    plan.table = torch.zeros_like(plan.table)
    c = new_cache(plan, H, D, cache)
    q = randn(new, H, D, seed=9)
    out = attend(plan, q, c)
    k, v = (x[0].double() * (1.0 if s is None else s[0].double()[..., None]) for x, s in ((c[0], c[2]), (c[1], c[3])))
    pos = torch.arange(ctx - new, ctx, device="cuda")
    times = (pos // P)[:, None] + (torch.arange(P, device="cuda") <= (pos % P)[:, None])
    score = torch.einsum("nhd,hjd->nhj", q.double(), k) * D ** -0.5
    p = torch.softmax(score + torch.log(times.double())[:, None], -1)
    want, mass = torch.einsum("nhj,hjd->nhd", p, v), torch.einsum("nhj,hjd->nhd", p, v.abs())
    size = float((torch.einsum("nhd,hjd->nhj", q.double().abs(), k.abs()) * D ** -0.5).max())
    # beside the usual bound: fp32 sums of millions of terms, added in an order of at most 2^17 partial sums a row
    bound = attention_bound(want, mass, size, F16, D, 0, 0.0) + 2.0 ** 17 * 2.0 ** -24 * mass
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())
    assert K.device_error() == 0


# ---- logits ----------------------------------------------------------------------------------------------------------

def logits_case(B, V, dtype, L=0, m=0, mask=False, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    x = torch.empty((B, V + pad), dtype=dtype, device="cuda")[:, :V]
    x.copy_(torch.randn((B, V), generator=g, device="cuda") * 3)
    kw = {}
    if L:
        kw["history"] = (r(B, L) ** 2 * V * 1.02).int() - 1  # some ids on either side of the vocabulary
        kw["history_len"] = torch.randint(0, L + 3, (B,), generator=g, device="cuda", dtype=torch.int32)
        kw["prompt_len"] = torch.randint(-1, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        kw.update(repetition=1 + r(B), frequency=r(B) - 0.3, presence=r(B))
    if m:
        kw["bias_ids"] = torch.randint(-2, min(V, 50) + 1, (B, m), generator=g, device="cuda", dtype=torch.int32)
        kw["bias"] = r(B, m) * 4 - 2
    if mask:
        kw["mask"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32 + 1), generator=g, device="cuda", dtype=torch.int64).int()
    return x, kw


def check_logits(x, kw, got):
    want, size = logits_64(x, **kw)
    inf = torch.isinf(want)
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got) & (got < 0), inf & (want < 0))
    # a product, two penalties and the biases, each rounded to 32 bits, of values that sum to at most `size`; then the type
    ops = 6 + (kw["bias"].shape[1] if "bias" in kw else 0)
    bound = size * ops * 2.0 ** -24 + want.abs().nan_to_num(0, 0, 0) * torch.finfo(x.dtype).eps / 2 + 2.0 ** -25
    err = (got - want).abs()[~inf]
    assert (err <= bound[~inf]).all(), float((err - bound[~inf]).max())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,V,L,m,mask,pad", [(1, 50257, 300, 16, True, 7), (3, 50257, 0, 0, True, 0), (2, 1, 5, 2, True, 0), (5, 31, 9, 0, False, 0), (4, 33, 700, 70, True, 1),
                                              (2, 4096, 64, 3, False, 0), (2, 4097, 1, 1, True, 0), (7, 8193, 5000, 200, True, 7), (3, 1000, 0, 33, False, 4), (300, 517, 20, 5, True, 3)])
def test_logits(B, V, L, m, mask, pad, dtype):
    x, kw = logits_case(B, V, dtype, L, m, mask, pad=pad)
    keep = x.clone()
    got = K.logits_process(x, **kw)
    check_logits(keep, kw, got)
    assert same(x, keep)
    # the parts alone, and in place
    for names in (["mask"], ["bias_ids", "bias"], ["history", "repetition"], ["history", "history_len", "frequency"], ["history", "prompt_len", "presence"], []):
        if all(n in kw for n in names):
            part = {n: kw[n] for n in names}
            y = x.clone() if not pad else torch.cat([x, x[:, :1]], 1)[:, :V]
            assert K.logits_process(y, **part, out=y) is y
            check_logits(keep, part, y)
    assert same(got, K.logits_process(x, **kw))


def test_logits_that_are_not_numbers_and_rows_without_a_token():
    x, kw = logits_case(4, 300, F32, 40, 5, True)
    x[0, :7], x[1, 3], x[1, 4] = float("nan"), float("inf"), float("-inf")
    kw["mask"][2] = 0
    got, want = K.logits_process(x, **kw).cpu(), logits_64(x, **kw)[0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and (got[2] == float("-inf")).all()


def test_biases_of_one_token_add_in_order():
    # many entries for one token, large and small: in 32 bits the sum depends on the order, which is the list's
    x = torch.zeros((1, 64), device="cuda")
    ids = torch.full((1, 500), 5, dtype=torch.int32, device="cuda")
    ids[0, ::7] = 6
    b = randn(1, 500, dtype=F32) * 10 ** randn(1, 500, dtype=F32, seed=1)
    got = K.logits_process(x, bias_ids=ids, bias=b)
    for token in (5, 6):
        s = torch.zeros((), dtype=F32)
        for v in b[ids == token].cpu():
            s = s + v
        assert got[0, token].item() == s.item()


# ---- a run of them together --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache,dtype", [(F16, F16), (I8, BF16)])
def test_a_prompt_in_chunks_then_tokens_one_by_one(cache, dtype):
    """What each step attends to is what all steps before it stored: the same as attention over the whole at once."""
    D, P, H = 64, 16, 3
    total = [90, 41, 7]
    whole = Plan(total, total, P)
    q, k, v = (randn(whole.rows, H, D, dtype=dtype, seed=s) for s in (1, 2, 3))
    c = new_cache(whole, H, D, cache, fill=0)
    done = [0, 0, 0]
    for step in ([50, 41, 0], [30, 0, 3], [9, 0, 3], [1, 0, 1]):
        plan = Plan(step, [d + s for d, s in zip(done, step)], P)
        plan.table, plan.table_list, plan.width, plan.pages = whole.table, whole.table_list, whole.width, whole.pages
        rows = torch.cat([torch.arange(whole.starts[b] + done[b], whole.starts[b] + done[b] + step[b]) for b in range(3)]).cuda()
        K.kv_write(k[rows], v[rows], c[0], c[1], plan.q_start, plan.ctx_len, plan.table, c[2], c[3])
        check(plan, attend(plan, q[rows], c), q[rows], c)
        done = plan.ctx
    back = K.kv_read(c[0], c[1], whole.kv_start, whole.table, whole.rows, c[2], c[3], out_dtype=dtype)
    if cache == F16:
        assert same(back[0], k) and same(back[1], v)
    else:
        qk, s = quantised(k)
        assert same(back[0].cpu(), (qk.float() * s[..., None]).to(dtype))


def test_a_captured_step_follows_the_plan_in_memory_and_side_streams_work():
    D, P, H, B = 64, 16, 4, 5
    final = Plan([1] * B, [60 + 20 * b for b in range(B)], P)
    c = new_cache(final, H, D, F16)
    x = randn(B, 3, H, D)
    hist = torch.randint(0, 500, (B, 64), device="cuda", dtype=torch.int32)
    logits = randn(B, 500)
    lens = final.ctx_len.clone()
    out, shaped = torch.empty((B, H, D), dtype=F16, device="cuda"), torch.empty_like(logits)

    def step():
        K.kv_write(x[:, 1], x[:, 2], c[0], c[1], final.q_start, lens, final.table)
        K.paged_attention(x[:, 0], c[0], c[1], final.q_start, lens, final.table, out=out)
        K.logits_process(logits, hist, history_len=lens, frequency=torch_freq, out=shaped)

    torch_freq = torch.rand(B, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for back in (40, 17, 0):
        lens.copy_(final.ctx_len - back)
        x.copy_(randn(B, 3, H, D, seed=back + 1))
        graph.replay()
        plan = Plan([1] * B, [n - back for n in final.ctx], P)
        plan.table, plan.table_list, plan.width, plan.pages = final.table, final.table_list, final.width, final.pages
        check(plan, out, x[:, 0], c)
        check_logits(logits, dict(history=hist, history_len=lens, frequency=torch_freq), shaped)
        for b in range(B):
            page, slot = plan.places(b, [plan.ctx[b] - 1])[0]
            assert same(c[0][page, :, slot], x[b, 1]) and same(c[1][page, :, slot], x[b, 2])


FIRST_CALLS = """
import sys, torch
sys.path[:0] = sys.argv[1:]
from generation import Plan, new_cache
from pequegrad_b200 import kernels as K
work = []
for new, cache in (([1, 1], torch.float16), ([40, 90], torch.int8), ([300], torch.float16)):
    plan = Plan(new, [n + 50 for n in new], 16)
    c, x = new_cache(plan, 2, 64, cache), torch.randn((plan.rows, 3, 2, 64), device="cuda").half()
    work.append((plan, c, x, torch.empty((plan.rows, 2, 64), dtype=torch.float16, device="cuda")))
logits = torch.randn((2, 77), device="cuda")
shaped = torch.empty_like(logits)
read = [torch.empty((work[0][0].kv_starts[-1], 2, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
def step():
    for p, c, x, o in work:
        K.kv_write(x[:, 1], x[:, 2], c[0], c[1], p.q_start, p.ctx_len, p.table, c[2], c[3])
        K.paged_attention(x[:, 0], c[0], c[1], p.q_start, p.ctx_len, p.table, None, c[2], c[3], out=o)
    p, c = work[0][:2]
    K.kv_read(c[0], c[1], p.kv_start, p.table, read[0].shape[0], out=read)
    K.logits_process(logits, bias_ids=p.table[:, :1].contiguous(), bias=torch.ones((2, 1), device="cuda"), out=shaped)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
replayed = [t.clone() for t in [w[3] for w in work] + read + [shaped]]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(replayed, [w[3] for w in work] + read + [shaped])) and K.device_error() == 0
print("same")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(root), str(root / "tests")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


def test_operands_on_two_devices_are_refused():
    plan = Plan([1], [5], 16)
    c = new_cache(plan, 1, 64, F16)
    x = randn(1, 1, 64)
    with pytest.raises(ValueError, match="one device"):
        K.kv_write(x, x, c[0], c[1], plan.q_start.cpu(), plan.ctx_len, plan.table)
    with pytest.raises(ValueError, match="one device"):
        K.logits_process(randn(1, 8), mask=torch.zeros((1, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="does not have the rows"):
        K.kv_read(c[0], c[1], plan.kv_start, plan.table, 5, out=(x, x))
