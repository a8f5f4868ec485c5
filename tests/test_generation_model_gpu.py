"""GPT-2 over the paged cache: prompts, chunks and single tokens against the CPU restatement that sees whole sequences."""
import numpy as np
import pytest
import torch

from pequegrad_b200 import gpt2 as G
from pequegrad_b200 import kernels as K

pytestmark = pytest.mark.gpu

CFG = G.GPT2Config(n_layer=2, n_head=2, n_embd=128, vocab_size=517, block_size=300)


@pytest.fixture(scope="module")
def setup():
    w = G.init_weights(CFG, seed=5)
    rng = np.random.default_rng(6)
    for i in range(CFG.n_layer):
        for k, v in w[f"h{i}"].items():
            if k.endswith("_b"):
                w[f"h{i}"][k] = (rng.standard_normal(v.shape) * 0.02).astype(np.float32)
    # larger projections than the benchmark's, so that attention has a say in the logits
    for i in range(CFG.n_layer):
        w[f"h{i}"]["attn_w"] *= 8
    return w, G.GPT2(CFG, w)


def reference(w, tokens):
    return torch.from_numpy(G.reference_forward(CFG, w, np.array([tokens])))[0]


def quantised_reference(w, tokens):
    """The same with keys and values rounded as an int8 cache rounds them."""
    r = G.round_weights_fp16(w)
    C, H, T = CFG.n_embd, CFG.n_head, len(tokens)
    ln = lambda t, g, b: torch.nn.functional.layer_norm(t, (C,), g, b, 1e-5)  # noqa: E731

    def cached(t):
        s = t.abs().amax(-1, keepdim=True).clamp(min=1e-6) / 127
        return torch.round(t / s).clamp(-127, 127) * s

    x = r["wte"][torch.tensor(tokens)] + r["wpe"][:T]
    gone = torch.ones(T, T, dtype=torch.bool).triu(1)
    for i in range(CFG.n_layer):
        h = r[f"h{i}"]
        q, k, v = ((ln(x, h["ln1_g"], h["ln1_b"]) @ h["attn_w"] + h["attn_b"]).view(T, 3, H, C // H).permute(1, 2, 0, 3))
        s = (q @ cached(k).transpose(1, 2) / (C // H) ** 0.5).masked_fill(gone, float("-inf"))
        y = (torch.softmax(s, -1) @ cached(v)).transpose(0, 1).reshape(T, C)
        x = x + y @ h["proj_w"] + h["proj_b"]
        m = ln(x, h["ln2_g"], h["ln2_b"]) @ h["fc_w"] + h["fc_b"]
        x = x + torch.nn.functional.gelu(m, approximate="tanh") @ h["fc2_w"] + h["fc2_b"]
    return ln(x, r["lnf_g"], r["lnf_b"]) @ r["lm_head"]


def rounding(w, tokens, dtype):
    """How far the logits may move because an int8 cache rounds keys and values. The restatement with rounding against the one
    without says what half a step on every value does. The model rounds values that 16 bits have already moved, so its half
    steps fall otherwise but are no larger; the effect is a sum over thousands of them, of the same size: twice it bounds it."""
    return 2 * (quantised_reference(w, tokens) - reference(w, tokens)).abs().max().item() if dtype == torch.int8 else 0.0


def close(got, want, what, more=0.0):
    """The tolerance of the whole-sequence forward (16-bit weights and activations): 2e-2 of the largest logit."""
    assert got.shape == want.shape
    err = (got.float().cpu() - want).abs().max().item()
    assert err <= 2e-2 * max(1.0, want.abs().max().item()) + more, f"{what}: {err}"
    assert K.device_error() == 0


@pytest.mark.parametrize("dtype,page_size", [(None, 16), (torch.int8, 32)])
def test_cached_steps_match_the_whole_sequence(setup, dtype, page_size):
    w, model = setup
    rng = np.random.default_rng(3)
    total = [290, 150, 33]
    tokens = [rng.integers(0, CFG.vocab_size, n).tolist() for n in total]
    want = [reference(w, t) for t in tokens]
    more = max(rounding(w, t, dtype) for t in tokens)
    cache = model.new_cache(600, page_size, dtype)
    seqs = [cache.open() for _ in total]
    done = [0, 0, 0]
    # whole prompts, a chunk behind a context beside a single token, single tokens
    for step in ([200, 100, 30], [80, 1, 0], [1, 40, 1], [1, 1, 1], [1, 1, 1]):
        live = [b for b in range(3) if step[b]]
        plan = cache.extend([seqs[b] for b in live], [step[b] for b in live])
        ids = torch.tensor([t for b in live for t in tokens[b][done[b]:done[b] + step[b]]], dtype=torch.int32, device="cuda")
        every = model.forward_cached(ids, cache, plan, last_only=False)
        close(every, torch.cat([want[b][done[b]:done[b] + step[b]] for b in live]), f"step {step}", more)
        for b in live:
            done[b] += step[b]
    # the last rows alone
    plan = cache.extend([seqs[0], seqs[2]], [2, 0 + 1]) if done[2] < total[2] else cache.extend([seqs[0]], [2])
    live = [0, 2] if done[2] < total[2] else [0]
    n = [2, 1][: len(live)]
    ids = torch.tensor([t for b, k in zip(live, n) for t in tokens[b][done[b]:done[b] + k]], dtype=torch.int32, device="cuda")
    last = model.forward_cached(ids, cache, plan)
    close(last, torch.stack([want[b][done[b] + k - 1] for b, k in zip(live, n)]), "last rows", more)
    with pytest.raises(ValueError, match="one token id per row"):
        model.forward_cached(ids[:1], cache, cache.extend([seqs[1]], [2]))


def test_what_a_cache_holds_can_move_to_another(setup):
    """Read back from an int8 cache, written to a 16-bit one: the next token sees the same."""
    w, model = setup
    tokens = np.random.default_rng(4).integers(0, CFG.vocab_size, 70).tolist()
    up = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    old, new = model.new_cache(128, 16, torch.int8), model.new_cache(128, 64)
    a, b = old.open(), new.open()
    model.forward_cached(up(tokens[:-1]), old, old.extend([a], [69]))
    plan = new.extend([b], [69])
    for layer in range(CFG.n_layer):
        k, v = old.read(layer, [a], out_dtype=torch.float16)
        assert k.shape == (69, CFG.n_head, 64)
        new.write(layer, k, v, plan)
        for got, want in zip(new.read(layer, [b]), (k, v)):
            assert torch.equal(got, want)
    one = [model.forward_cached(up(tokens[-1:]), c, c.extend([s], [1])) for c, s in ((old, a), (new, b))]
    for logits in one:
        close(logits, reference(w, tokens)[-1:], "next token", rounding(w, tokens, torch.int8))


def shaped(logits, prompt, made, repetition, frequency, presence, bias, allowed):
    x = logits.double().clone()
    for t in set(prompt + made):
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    for t in set(made):
        x[t] -= frequency * made.count(t) + presence
    for t, v in bias.items():
        x[t] += v
    if allowed is not None:
        x[[t for t in range(len(x)) if t not in allowed]] = float("-inf")
    return x


@pytest.mark.parametrize("kw", [dict(), dict(repetition=1.4, frequency=0.3, presence=0.2, bias={5: 1.5, 77: -2.0}), dict(cache_dtype=torch.int8, page_size=32, repetition=1.2),
                                dict(mask=True, presence=0.5)])
def test_generated_tokens_are_the_best_ones(setup, kw):
    """Every pick is, by the CPU restatement's shaped logits, within twice the forward's tolerance of the best."""
    w, model = setup
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, CFG.vocab_size, n).tolist() for n in (40, 3, 17)]
    allowed = set(range(0, CFG.vocab_size, 3)) if kw.get("mask") else None
    call = dict(kw)
    if allowed is not None:
        words = torch.zeros((CFG.vocab_size + 31) // 32 * 32, dtype=torch.int64)
        words[sorted(allowed)] = 1
        words = (words.view(-1, 32) << torch.arange(32)).sum(1)
        row = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
        call["mask"] = lambda made: row.expand(len(made), -1).contiguous().cuda()
    out = model.generate(prompts, 12, **call)
    assert [len(t) for t in out] == [12] * 3
    for p, made in zip(prompts, out):
        want = reference(w, p + made)
        tol = (4e-2 * max(1.0, want.abs().max().item()) + 2 * rounding(w, p + made, kw.get("cache_dtype"))) * kw.get("repetition", 1.0)
        for i, t in enumerate(made):
            x = shaped(want[len(p) + i - 1], p, made[:i], kw.get("repetition", 1.0), kw.get("frequency", 0.0), kw.get("presence", 0.0), kw.get("bias", {}), allowed)
            assert x[t] >= x.max() - tol, (i, t, float(x[t]), float(x.max()))
            assert allowed is None or t in allowed


def test_generation_ends_behind_eos_and_refuses_what_does_not_fit(setup):
    _, model = setup
    prompts = [[1, 2, 3], [4, 5]]
    free = model.generate(prompts, 6)
    eos = free[0][2]
    ended = model.generate(prompts, 6, eos=eos)
    assert ended[0] == free[0][: free[0].index(eos) + 1]
    assert ended[1] == (free[1][: free[1].index(eos) + 1] if eos in free[1] else free[1])
    assert model.generate([], 5) == [] and model.generate(prompts, 0) == [[], []]
    with pytest.raises(ValueError, match="block_size"):
        model.generate([[1] * 298], 3)
    with pytest.raises(ValueError, match="empty"):
        model.generate([[]], 3)
    with pytest.raises(RuntimeError, match="pages are needed"):
        cache = model.new_cache(16)
        cache.extend([cache.open()], [17])
