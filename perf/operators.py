"""The operators of token-by-token generation, as measured cases: a paged key / value cache (written, read back, kept in
16 bits or quantised to int8 as it is written), attention of new tokens over that cache, and the shaping of logits
before a token is picked.

`run` computes a case either in plain torch operations (`own` false) or through the framework's entry points
(`own` true). Terms:
  rows      new tokens of all sequences, packed one after another; those of sequence b are rows
            q_start[b] .. q_start[b + 1] - 1 and stand at the positions that end at ctx_len[b] - 1
  cache     [pages, kv heads, page size, head dim]; page_table[b, i] is the page of positions i * page size and up,
            -1 where there is none
  int8      one scale per cached token and head: max(max |x|, 1e-6) / 127, values rint(x / scale)
"""
import random

import torch

own = False

KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one step of a batch of GPT-2 sequences: each stores its newest token
        dict(name="write_step", op="write", B=32, new=1, ctx=1024, ragged=True, Hkv=12, D=64, P=16, dtype="f16", int8=False, mix=1),
        # prompts arrive at an int8 cache; what was stored is read back for another request
        dict(name="write_prompts_int8", op="write", B=8, new=500, ctx=1500, ragged=True, Hkv=8, D=128, P=32, dtype="bf16", int8=True, mix=2),
        # one short GPT-2 sequence moved out of its pages
        dict(name="read_one", op="read", B=1, ctx=777, ragged=False, Hkv=12, D=64, P=16, dtype="f16", int8=False, mix=3),
        # long int8 sequences expanded for a pass that wants them contiguous in 16 bits
        dict(name="read_long_int8", op="read", B=12, ctx=8192, ragged=True, Hkv=8, D=128, P=64, dtype="bf16", int8=True, mix=4),
        # the latency of one token of one GPT-2 sequence
        dict(name="decode_one", op="attention", B=1, new=1, ctx=1000, ragged=False, Hq=12, Hkv=12, D=64, P=16, dtype="f16", int8=False, mix=5),
        # a serving step of GPT-2, contexts of all lengths
        dict(name="decode_batch", op="attention", B=64, new=1, ctx=1024, ragged=True, Hq=12, Hkv=12, D=64, P=16, dtype="f16", int8=False, mix=6),
        # long contexts, grouped heads, int8 cache
        dict(name="decode_long_int8", op="attention", B=16, new=1, ctx=32768, ragged=True, Hq=32, Hkv=8, D=128, P=64, dtype="bf16", int8=True, mix=7),
        # whole GPT-2 prompts, no context before them
        dict(name="prompts", op="attention", B=8, new=1024, ctx=1024, ragged=False, Hq=12, Hkv=12, D=64, P=16, dtype="f16", int8=False, mix=8),
        # chunks of long prompts behind what is already cached
        dict(name="chunk_grouped", op="attention", B=4, new=512, ctx=8000, ragged=True, Hq=32, Hkv=8, D=128, P=64, dtype="bf16", int8=False, mix=9),
        # the same over an int8 cache, odd sizes
        dict(name="chunk_int8", op="attention", B=2, new=301, ctx=5003, ragged=True, Hq=12, Hkv=12, D=64, P=32, dtype="f16", int8=True, mix=10),
        # one row of GPT-2 logits before greedy choice
        dict(name="logits_one", op="logits", B=1, V=50257, L=300, bias=16, mask=True, dtype="f16", mix=11),
        # a large serving batch, long histories
        dict(name="logits_batch", op="logits", B=256, V=50257, L=2000, bias=64, mask=True, dtype="f16", mix=12),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "attention", "logits"])
    dtype, mix = rng.choice(["f16", "bf16"]), rng.randrange(1 << 20)
    if op == "logits":
        V = _log(rng, 200, 60000)
        return dict(op=op, B=_log(rng, 1, max(1, min(256, 6_000_000 // V))), V=V, L=_log(rng, 1, 4000), bias=rng.choice([0, 1, 16, 100, 300]),
                    mask=rng.random() < 0.7, dtype=rng.choice(["f16", "bf16", "f32"]), mix=mix)
    Hq, Hkv = rng.choice([(12, 12), (16, 16), (32, 8), (16, 2), (28, 4), (8, 1), (6, 2)])
    cache = dict(Hkv=Hkv, D=rng.choice([64, 128]), P=rng.choice([16, 32, 64, 128]), dtype=dtype, int8=rng.random() < 0.5, ragged=rng.random() < 0.8, mix=mix)
    token = Hkv * cache["D"]  # cached values of one token, of K as of V
    if op == "read":
        ctx = _log(rng, 1, 16384)
        return dict(op=op, B=_log(rng, 1, max(1, min(64, 50_000_000 // (ctx * token)))), ctx=ctx, **cache)
    if op == "write":
        new = rng.choice([1, 1, _log(rng, 2, 2000)])
        ctx = new + rng.choice([0, _log(rng, 1, 1000)])
        return dict(op=op, B=_log(rng, 1, max(1, min(128, 8_000_000 // (ctx * token)))), new=new, ctx=ctx, **cache)
    if rng.random() < 0.5:  # a step: one token, or the few of a speculated continuation
        new = rng.choice([1, 1, 1, 2, 5])
        ctx = new + _log(rng, 1, 30000)
        return dict(op=op, B=_log(rng, 1, max(1, min(128, 60_000_000 // (ctx * token)))), new=new, ctx=ctx, Hq=Hq, **cache)
    new = _log(rng, 6, 1500)
    ctx = new + rng.choice([0, _log(rng, 1, max(1, min(8000, 180_000_000 // (new * Hq))))])
    return dict(op=op, B=_log(rng, 1, max(1, min(16, 200_000_000 // (new * ctx * Hq), 20_000_000 // (ctx * token)))), new=new, ctx=ctx, Hq=Hq, **cache)


def _lengths(c):
    """(new tokens, cached tokens) of each sequence; the second counts the first. They belong to the case, not to a seed."""
    r = random.Random(c["mix"])
    B, new, ctx = c["B"], c.get("new", 0), c["ctx"]
    if not c["ragged"]:
        return [new] * B, [ctx] * B
    n = [new if new <= 2 else r.randint(max(1, new // 3), new) for _ in range(B)]
    return n, [r.randint(max(n[b], ctx // 4), ctx) if b else ctx for b in range(B)]


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, **dev)  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=g, **dev)  # noqa: E731
    c, dt = case, KINDS[case["dtype"]]
    if c["op"] == "logits":
        B, V, L = c["B"], c["V"], c["L"]
        r = random.Random(c["mix"])
        total = [L] + [r.randint(1, L) for _ in range(B - 1)]
        rows = torch.empty((B, (V + 7) // 8 * 8), dtype=dt, **dev)  # rows padded as the GPT-2 head writes them
        logits = rows[:, :V]
        logits.copy_(randn(B, V) * 3)
        # text repeats itself: few tokens often, most of them rarely
        history = (torch.rand((B, L), generator=g, **dev) ** 3 * V).to(torch.int32).clamp_(max=V - 1)
        s = dict(logits=logits, history=history, total=i32(total), prompt=i32([t // 2 for t in total]),
                 repetition=1 + torch.rand(B, generator=g, **dev) * 0.3, frequency=torch.rand(B, generator=g, **dev) * 0.5,
                 presence=torch.rand(B, generator=g, **dev) * 0.5, out=torch.empty_like(logits), bias_ids=None, bias=None, mask=None)
        if c["bias"]:
            s["bias_ids"] = torch.randint(0, V, (B, c["bias"]), generator=g, dtype=torch.int32, **dev)
            s["bias"] = randn(B, c["bias"]) * 2
        if c["mask"]:  # bit v % 32 of word v // 32: token v may follow. Most rows of a grammar allow little.
            words = torch.randint(-(1 << 31), 1 << 31, (B, (V + 31) // 32), generator=g, dtype=torch.int64, **dev)
            s["mask"] = words.to(torch.int32)
        return dict(case=c, **s)
    B, H, D, P = c["B"], c["Hkv"], c["D"], c["P"]
    new, ctx = _lengths(c)
    need = [-(-x // P) for x in ctx]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, **dev).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, **dev)
    at = _starts(need)
    for b in range(B):
        table[b, :need[b]] = order[at[b]:at[b + 1]]
    s = dict(table=table, ctx=i32(ctx), q_start=i32(_starts(new)), kv_start=i32(_starts(ctx)), rows=sum(ctx), k_scale=None, v_scale=None)
    shape = (pages, H, P, D)
    if c["int8"]:
        for n in ("k", "v"):
            s[n + "_cache"] = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, **dev)
            s[n + "_scale"] = (0.5 + torch.rand(shape[:3], generator=g, **dev)) * (2.5 / 127)
    else:
        for n in ("k", "v"):
            s[n + "_cache"] = torch.randn(shape, generator=g, dtype=dt, **dev)
    R = sum(new)
    if c["op"] == "write":  # the keys and values of a packed projection
        kv = randn(R, 2, H, D).to(dt)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
    elif c["op"] == "attention":
        s["q"] = randn(R, c["Hq"], D).to(dt)
    return dict(case=c, **s)


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _row_places(s):
    """For every row: its sequence, its position there, and the page and slot of that position."""
    R, P = int(s["k"].shape[0]), s["case"]["P"]
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:], torch.arange(R, device="cuda"), right=True)
    pos = s["ctx"].long()[seq] - (start[seq + 1] - start[seq]) + torch.arange(R, device="cuda") - start[seq]
    return seq, pos, s["table"].long()[seq, pos // P], pos % P


def _cached_places(s):
    """The same for every cached token, sequence after sequence."""
    P = s["case"]["P"]
    start, r = s["kv_start"].long(), torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(start[1:], r, right=True)
    pos = r - start[seq]
    return s["table"].long()[seq, pos // P], pos % P


def _plain_read(s):
    page, slot = _cached_places(s)
    out = []
    for n in ("k", "v"):
        x = s[n + "_cache"][page, :, slot]
        if s["k_scale"] is not None:
            x = (x.float() * s[n + "_scale"][page, :, slot][..., None]).to(KINDS[s["case"]["dtype"]])
        out.append(x)
    return out


def _plain_write(s):
    _, _, page, slot = _row_places(s)
    for n in ("k", "v"):
        x = s[n]
        if s["k_scale"] is not None:
            scale = x.float().abs().amax(-1).clamp(min=1e-6) / 127
            x = torch.round(x.float() / scale[..., None]).clamp(-127, 127).to(torch.int8)
            s[n + "_scale"][page, :, slot] = scale
        s[n + "_cache"][page, :, slot] = x
    return _plain_read(s) if s["k_scale"] is not None else [s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    c = s["case"]
    B, D, P, Hkv, G = c["B"], c["D"], c["P"], c["Hkv"], c["Hq"] // c["Hkv"]
    q, start, ctx = s["q"], s["q_start"].long(), s["ctx"].long()
    n = start[1:] - start[:-1]
    width = int(s["table"].shape[1]) * P
    page = s["table"].long().clamp(min=0)

    def cached(x, scale):  # [B, Hkv, width, ...] in 32 bits
        x = x[page].float()
        x = x if scale is None else x * scale[page][..., None]
        return x.transpose(1, 2).reshape(B, Hkv, width, D)

    k, v = cached(s["k_cache"], s["k_scale"]), cached(s["v_cache"], s["v_scale"])
    most = max(_lengths(c)[0])
    i = torch.arange(most, device="cuda")
    row = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[row].float().reshape(B, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * most, D)
    score = (qp @ k.transpose(-1, -2) * D ** -0.5).reshape(B, Hkv, G, most, width)
    last = (ctx - n)[:, None] + i  # the position of each row
    seen = torch.arange(width, device="cuda") <= last[..., None]  # [B, most, width]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(B, Hkv, G * most, width)
    o = (p @ v).reshape(B, Hkv, G, most, D).permute(0, 3, 1, 2, 4).reshape(B, most, c["Hq"], D)
    r = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], r, right=True)
    return o[seq, r - start[seq]].to(q.dtype)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    at = torch.arange(s["history"].shape[1], device="cuda")
    there = (at < s["total"][:, None]).int()
    made = there * (at >= s["prompt"][:, None]).int()
    ids = s["history"].long()
    seen = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, ids, there) > 0
    count = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, ids, made)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + torch.zeros((B, V), device="cuda").scatter_add_(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        x = x.masked_fill((s["mask"][:, v // 32] >> (v % 32)) & 1 == 0, float("-inf"))
    return x.to(s["logits"].dtype)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from pequegrad_b200 import kernels as K
        cache = (s["k_cache"], s["v_cache"]) if op != "logits" else ()
        scales = dict(k_scale=s["k_scale"], v_scale=s["v_scale"]) if op != "logits" else {}
        if op == "write":
            K.kv_write(s["k"], s["v"], *cache, s["q_start"], s["ctx"], s["table"], **scales)
            if s["k_scale"] is None:
                return list(cache)
        if op in ("write", "read"):
            return list(K.kv_read(*cache, s["kv_start"], s["table"], s["rows"], out_dtype=KINDS[s["case"]["dtype"]], **scales))
        if op == "attention":
            return K.paged_attention(s["q"], *cache, s["q_start"], s["ctx"], s["table"], **scales)
        return K.logits_process(s["logits"], history=s["history"], history_len=s["total"], prompt_len=s["prompt"], repetition=s["repetition"],
                                frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], out=s["out"])
    return {"write": _plain_write, "read": _plain_read, "attention": _plain_attention, "logits": _plain_logits}[op](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "logits":
        r = random.Random(c["mix"])
        tokens = c["L"] + sum(r.randint(1, c["L"]) for _ in range(c["B"] - 1))
        return {"bytes": c["B"] * (c["V"] * 2 * es + c["bias"] * 8 + (c["V"] // 8 if c["mask"] else 0)) + tokens * 4, "flops": 0}
    new, ctx = _lengths(c)
    D, Hkv = c["D"], c["Hkv"]
    held = Hkv * ((D + 4) if c["int8"] else D * es)  # one cached token, of K as of V
    plain = Hkv * D * es
    if c["op"] == "write":
        return {"bytes": 2 * sum(new) * (plain + held) + (2 * sum(ctx) * (plain + held) if c["int8"] else 0), "flops": 0}
    if c["op"] == "read":
        return {"bytes": 2 * sum(ctx) * (plain + held), "flops": 0}
    pairs = sum(n * x - n * (n - 1) // 2 for n, x in zip(new, ctx))
    return {"bytes": 2 * sum(ctx) * held + 2 * sum(new) * c["Hq"] * D * es, "flops": 4 * D * c["Hq"] * pairs}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------------

def _exact_sequence(s, b, n, name):
    """Sequence b's first n cached tokens, [n, Hkv, D] in 64 bits."""
    P = s["case"]["P"]
    pages = s["table"][b, : -(-n // P)].long()
    x = s[name + "_cache"].index_select(0, pages).double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"].index_select(0, pages).double().unsqueeze(-1)
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:n]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "logits":
        rows = []
        for b in range(c["B"]):
            x = s["logits"][b].double()
            total, prompt = int(s["total"][b]), int(s["prompt"][b])
            past = s["history"][b, :total].long()
            met, made = torch.bincount(past, minlength=c["V"]), torch.bincount(past[prompt:], minlength=c["V"])
            rep, freq, pres = (float(s[n][b]) for n in ("repetition", "frequency", "presence"))
            x = torch.where(met > 0, x * torch.where(x > 0, 1 / rep, rep), x) - freq * made - pres * made.clamp(max=1)
            if c["bias"]:
                x.index_add_(0, s["bias_ids"][b].long(), s["bias"][b].double())
            if c["mask"]:
                bits = torch.arange(32, device="cuda", dtype=torch.int32)
                allowed = (s["mask"][b][:, None] >> bits & 1).flatten()[: c["V"]].bool()
                x[~allowed] = float("-inf")
            rows.append(x)
        return torch.stack(rows)
    new, ctx = _lengths(c)
    P, at = c["P"], _starts(new)
    if c["op"] == "write":
        for n in ("k", "v"):
            for b in range(c["B"]):
                x = s[n][at[b]:at[b + 1]]
                pos = torch.arange(ctx[b] - new[b], ctx[b], device="cuda")
                page, slot = s["table"][b].long()[pos // P], pos % P
                if c["int8"]:
                    # the scale is a 32-bit number, and the quotient is taken in 32 bits: 64 bits rounded once more give just that
                    scale = (x.double().abs().amax(-1).clamp(min=1e-6) / 127).float()
                    x = (x.double() / scale.double()[..., None]).float().round().clamp(-127, 127).to(torch.int8)
                    s[n + "_scale"].index_put_((page[:, None], torch.arange(c["Hkv"], device="cuda"), slot[:, None]), scale)
                s[n + "_cache"].index_put_((page[:, None], torch.arange(c["Hkv"], device="cuda"), slot[:, None]), x)
        if not c["int8"]:
            return [s["k_cache"].double(), s["v_cache"].double()]
    if c["op"] in ("write", "read"):
        return [torch.cat([_exact_sequence(s, b, ctx[b], n) for b in range(c["B"])]) for n in ("k", "v")]
    outs, G = [], c["Hq"] // c["Hkv"]
    for b in range(c["B"]):
        k, v = (_exact_sequence(s, b, ctx[b], n).transpose(0, 1) for n in ("k", "v"))
        q = s["q"][at[b]:at[b + 1]].double()
        heads = []
        for h in range(c["Hq"]):
            score = q[:, h] @ k[h // G].T / c["D"] ** 0.5
            score += torch.full_like(score, float("-inf")).triu(ctx[b] - new[b] + 1)
            heads.append(torch.softmax(score, -1) @ v[h // G])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
