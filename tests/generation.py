"""Plans, caches and plain 64-bit forms for the tests of the paged cache, the attention over it and the logit shaping."""
from __future__ import annotations

import torch


class Plan:
    """Packed rows of sequences with `new` new and `ctx` cached tokens each, over shuffled pages."""

    def __init__(self, new, ctx, P, device="cuda", seed=0, pad_rows=0, spare_pages=2, spare_width=1):
        g = torch.Generator().manual_seed(seed)
        self.new, self.ctx, self.P, self.device = list(new), list(ctx), P, device
        need = [-(-max(c, 0) // P) for c in ctx]
        self.pages = sum(need) + spare_pages
        order = torch.randperm(self.pages, generator=g).tolist()
        self.width = max(need, default=0) + spare_width
        self.table_list = []
        for n in need:
            self.table_list.append([order.pop() for _ in range(n)] + [-1] * (self.width - n))
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.kv_starts = [0]
        for c in ctx:
            self.kv_starts.append(self.kv_starts[-1] + c)
        self.rows = self.starts[-1] + pad_rows
        i32 = lambda x, shape=None: torch.tensor(x, dtype=torch.int32, device=device) if x else torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        self.q_start, self.ctx_len, self.kv_start = i32(self.starts), i32(self.ctx, (0,)), i32(self.kv_starts)
        self.table = i32(self.table_list, (0, self.width))

    def places(self, b, positions):
        """(page, slot) of positions of sequence b; page None where there is none."""
        out = []
        for p in positions:
            page = self.table_list[b][p // self.P] if 0 <= p and p // self.P < self.width else -1
            out.append((page if 0 <= page < self.pages else None, p % self.P))
        return out


def new_cache(plan, H, D, dtype, layout="hpd", fill=None, seed=1):
    """(k_cache, v_cache, k_scale, v_scale): random values, or `fill` everywhere; "phd" keeps heads inside the slots."""
    g = torch.Generator(device=plan.device).manual_seed(seed)
    shape = (plan.pages, H, plan.P, D) if layout == "hpd" else (plan.pages, plan.P, H, D)
    out = []
    for _ in range(2):
        if dtype == torch.int8:
            c = torch.randint(-127, 128, shape, generator=g, device=plan.device, dtype=torch.int8)
        else:
            c = torch.randn(shape, generator=g, device=plan.device).to(dtype)
        if fill is not None:
            c.fill_(fill)
        out.append(c if layout == "hpd" else c.permute(0, 2, 1, 3))
    if dtype != torch.int8:
        return out[0], out[1], None, None
    s = [(torch.rand((plan.pages, H, plan.P), generator=g, device=plan.device) + 0.5) / 50 for _ in range(2)]
    return out[0], out[1], s[0], s[1]


def gather(plan, b, n, cache, scale):
    """Sequence b's first n cached tokens [n, H, D] in 64 bits, and which of them have a page [n]."""
    H, D = cache.shape[1], cache.shape[3]
    out = torch.zeros((n, H, D), dtype=torch.float64, device=cache.device)
    there = torch.zeros(n, dtype=torch.bool)
    places = plan.places(b, range(n))
    idx = [i for i, (page, _) in enumerate(places) if page is not None]
    if idx:
        pg = torch.tensor([places[i][0] for i in idx], device=cache.device)
        sl = torch.tensor([places[i][1] for i in idx], device=cache.device)
        x = cache[pg, :, sl].double()
        if scale is not None:
            x = x * scale[pg, :, sl].double()[..., None]
        out[torch.tensor(idx, device=cache.device)] = x
        there[idx] = True
    return out, there.to(cache.device)


def attention_64(plan, q, cache, scale):
    """(out, sum of p |v|, largest sum of |q k| scale) of every row of the plan, in 64 bits; rows without a key are zero."""
    kc, vc, ks, vs = cache
    R, Hq, D = q.shape
    Hkv = kc.shape[1]
    G = Hq // Hkv
    out = torch.zeros((R, Hq, D), dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    size = 0.0
    for b, (n, c) in enumerate(zip(plan.new, plan.ctx)):
        c = min(c, plan.width * plan.P)
        if n == 0:
            continue
        k, there = gather(plan, b, max(c, 0), kc, ks)
        v, _ = gather(plan, b, max(c, 0), vc, vs)
        rows = slice(plan.starts[b], plan.starts[b] + n)
        pos = torch.arange(n, device=q.device) + plan.ctx[b] - n
        seen = (torch.arange(max(c, 0), device=q.device)[None] <= pos[:, None]) & there[None]
        # what a mask leaves out has no say, whatever it holds
        gone = ~seen.any(0)
        k = k.masked_fill(gone[:, None, None], 0)
        v = v.masked_fill(gone[:, None, None], 0)
        qq = q[rows].double().reshape(n, Hkv, G, D)
        s = torch.einsum("nhgd,chd->nhgc", qq, k) * scale
        if s.numel():
            size = max(size, float((torch.einsum("nhgd,chd->nhgc", qq.abs(), k.abs()) * scale).nan_to_num(0, 0, 0).max()))
        s = s.masked_fill(~seen[:, None, None], float("-inf"))
        p = torch.softmax(s, -1).masked_fill(~seen[:, None, None], 0) if s.numel() else s
        out[rows] = torch.einsum("nhgc,chd->nhgd", p, v).reshape(n, Hq, D)
        mass[rows] = torch.einsum("nhgc,chd->nhgd", p, v.abs()).reshape(n, Hq, D)
    return out, mass, size


def attention_bound(want, mass, size, dtype, D, keys, vmax):
    """How far a 16-bit result may be off. The result is rounded (half a step h of its value); each probability is rounded to
    16 bits before the second product (h of sum p |v|); probabilities carry the error of the fp32 scores (D + 8 roundings
    of terms that sum to `size`, in absolute terms of the exponent) and 1e-4 for the approximated exponential, in numerator
    and denominator. float16 drops what is below 2^-25 of a probability of one."""
    h = torch.finfo(dtype).eps / 2
    d = 1e-4 + (D + 8) * 2.0 ** -24 * size
    tiny = keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    return h * want.abs() + h * mass + d * (mass + want.abs()) + tiny + 2.0 ** -24


def quantised(x):
    """(q, scale) of [.., D] 16-bit values by the rule of the cache, in 32 bits on the CPU."""
    x = x.float().cpu()
    s = x.abs().amax(-1).clamp(min=1e-6) / 127
    bad = ~torch.isfinite(x).all(-1)
    q = torch.round(x / s[..., None]).clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q).to(torch.int8)
    return q, torch.where(bad, torch.full_like(s, float("nan")), s)


def logits_64(x, history=None, history_len=None, prompt_len=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias=None, mask=None):
    x = x.double().cpu()
    B, V = x.shape
    out = x.clone()
    size = x.abs()
    for r in range(B):
        if history is not None:
            n = min(max(int(history_len[r]), 0), history.shape[1]) if history_len is not None else history.shape[1]
            p = min(max(int(prompt_len[r]), 0), n) if prompt_len is not None else 0
            h = history[r].cpu().long()
            ok = lambda t: t[(t >= 0) & (t < V)]  # noqa: E731
            met, made = torch.bincount(ok(h[:n]), minlength=V), torch.bincount(ok(h[p:n]), minlength=V)
            if repetition is not None:
                rep = float(repetition[r])
                out[r] = torch.where(met > 0, torch.where(out[r] > 0, out[r] / rep, out[r] * rep), out[r])
                size[r] = torch.maximum(size[r], out[r].abs())
            f = float(frequency[r]) if frequency is not None else 0.0
            q = float(presence[r]) if presence is not None else 0.0
            out[r] -= f * made + q * (made > 0)
            size[r] += abs(f) * made + abs(q) * (made > 0)
        if bias_ids is not None:
            ids = bias_ids[r].cpu().long()
            keep = (ids >= 0) & (ids < V)
            out[r].index_add_(0, ids[keep], bias[r].cpu().double()[keep])
            size[r].index_add_(0, ids[keep], bias[r].cpu().double().abs()[keep])
        if mask is not None:
            bits = (mask[r].cpu()[:, None] >> torch.arange(32, dtype=torch.int32)) & 1
            out[r][bits.flatten()[:V] == 0] = float("-inf")
    return out, size
