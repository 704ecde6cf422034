"""Rules on logits and the choice of tokens, against the definition in 64 bits.

Adjusted logits: each of the operations is rounded by itself, half a step (2^-24) of its result; the bound adds up the magnitudes.
Chosen tokens: the reference works on the adjusted logits, so their order is exact.  A weight exp(-z), z < 32, is off by z 2^-23 from
the two roundings of z and two steps of the exponential, 4e-6 of it in all; sums add 1e-6.  SLACK = 1e-5 of the whole covers what that moves
at a border: a token is right if it is the one for some placing of the borders within it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
SLACK = 1e-5


@pytest.fixture(scope="module")
def ops():
    from inference_engine_b200 import ops

    return ops


def cuda(x, dtype=None):
    return torch.as_tensor(np.asarray(x)).to("cuda", dtype).contiguous()


# ----------------------------------------------------------------------------- references
def adjusted(l, rules):
    """(adjusted logits in 64 bits, bound) of rows under a Rules record of the library."""
    r = {k: None if v is None else (v.double() if v.is_floating_point() else v.long()).cpu().numpy()
         for k, v in vars(rules).items() if isinstance(v, torch.Tensor) or v is None}
    l = l.double().cpu().numpy().copy()
    E, V = l.shape
    size = np.abs(l)
    for e in range(E):
        slot = e if r["slots"] is None else r["slots"][e]
        if slot < 0:
            continue
        if r["history"] is not None:
            n = r["lengths"][e]
            h = r["history"][slot][:n]
            prompt = n if r["prompts"] is None else r["prompts"][e]
            out = np.bincount(h[prompt:], minlength=V)
            seen = np.bincount(h, minlength=V) > 0
            rep = 1.0 if r["repetition"] is None else r["repetition"][e]
            l[e][seen] = np.where(l[e][seen] > 0, l[e][seen] / rep, l[e][seen] * rep)
            size[e] += np.abs(l[e])
            for name, c in (("frequency", out), ("presence", out > 0)):
                if r[name] is not None:
                    l[e] -= r[name][e] * c
                    size[e] += 2 * np.abs(r[name][e]) * c
        if r["bias"] is not None:
            for i, b in zip(r["bias_ids"][e], r["bias"][e]):
                if i >= 0:
                    l[e][i] += b
                    size[e][i] += 3 * abs(b) + abs(l[e][i])
        if r["masks"] is not None and r["mask_rows"][e] >= 0:
            words = r["masks"][r["mask_rows"][e]].astype(np.int32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:V]
            l[e][bits == 0] = -np.inf
    return l, 6 * 2.0 ** -24 * size


def check_adjusted(got, l, rules):
    want, bound = adjusted(l, rules)
    got = got.double().cpu().numpy()
    idle = np.zeros(len(got), bool) if rules.slots is None else (rules.slots < 0).cpu().numpy()
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= bound
    assert (same | near)[~idle].all()


def check_choice(l, draw, tokens, logprobs):
    """l: adjusted logits, fp32."""
    l = l.double().cpu().numpy()
    l = np.where(np.isnan(l), -np.inf, l)
    num = lambda t, e, none: none if t is None else t[e].item()  # noqa: E731
    for e in range(len(l)):
        row, t, lp = l[e], int(tokens[e]), float(logprobs[e])
        m = row.max()
        if m == -np.inf:
            assert t == -1 and lp == -math.inf
            continue
        order = np.argsort(-row, kind="stable")
        with np.errstate(invalid="ignore"):
            behind = np.where(row == m, 0.0, m - row)
        ref = -behind[t] - math.log(np.exp(-behind).sum())
        assert abs(lp - ref) <= 5e-6 + 2.0 ** -22 * abs(ref), (e, lp, ref)
        tau, k, p = num(draw.temperature, e, 1.0), num(draw.top_k, e, 0), num(draw.top_p, e, 1.0)
        if not tau > 0 or k == 1:
            assert t == order[0], (e, t, order[0])
            continue
        w = np.exp(-behind / tau)
        first = order[:k] if k > 0 else order
        before = np.cumsum(w[first]) - w[first]
        total = w[first].sum()
        sets = []
        for s in (-SLACK, SLACK):
            keep = (before < (max(p, 0.0) + s) * total) | (p >= 1)
            keep &= w[first] * (1 + s) >= num(draw.min_p, e, 0.0)
            keep[0] = True
            kept = np.zeros_like(w)
            kept[first[keep]] = w[first[keep]]
            sets.append(kept)
        must, may = sets
        u = min(max(draw.uniform[e].item(), 0.0), 1.0)
        assert may[t] > 0, (e, t, "is not kept")
        assert must[:t].sum() <= u * may.sum() + SLACK * total, (e, t, "lies too far on")
        assert may[: t + 1].sum() >= u * must.sum() - SLACK * total, (e, t, "lies too far in front")


# ----------------------------------------------------------------------------- inputs
def make_rules(ops, E, V, longest, g, bias=5, masks=True, shuffle=True):
    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g) * (hi - lo) + lo

    lengths = (uniform(0, 1, E) ** 2 * (longest + 1)).int().clamp(max=longest)
    lengths[0] = longest
    history = (uniform(0, 1, E + 2, longest) ** 3 * V).int().clamp(max=V - 1)
    words = (V + 31) // 32 + 1
    bits = torch.randint(-(1 << 31), 1 << 31, (3, words), generator=g).int()
    ids = torch.randint(-1, V, (E, bias), generator=g).int()
    if bias > 2:
        ids[:, 2] = ids[:, 0]  # the same token twice
    off = torch.rand(E, generator=g) < 0.3
    return ops.Rules(
        history=cuda(history), slots=cuda((torch.randperm(E + 2, generator=g)[:E] if shuffle else torch.arange(E)), torch.int32), lengths=cuda(lengths),
        prompts=cuda((uniform(0, 1, E) * (lengths + 1)).int()), repetition=cuda(torch.where(off, torch.ones(E), uniform(0.7, 1.6, E))),
        presence=cuda(torch.where(off, torch.zeros(E), uniform(-0.5, 1, E))), frequency=cuda(torch.where(off, torch.zeros(E), uniform(-0.2, 0.8, E))),
        bias_ids=cuda(ids) if bias else None, bias=cuda(uniform(-6, 6, E, bias)) if bias else None,
        masks=cuda(bits) if masks else None, mask_rows=cuda(torch.randint(-1, 3, (E,), generator=g).int()) if masks else None)


def make_logits(E, V, dtype, g, pad=0, spread=3.0):
    l = torch.randn(E, V, generator=g) * spread
    l[:, torch.randint(0, V, (20,), generator=g)] += 8.0
    full = torch.full((E, V + pad), float("nan"))
    full[:, :V] = l
    return full.to("cuda", dtype)[:, :V]


def make_draw(ops, E, g, kind="mixed"):
    tau = 0.4 + torch.rand(E, generator=g) * 1.2
    k, p, m = torch.zeros(E, dtype=torch.int32), torch.ones(E), torch.zeros(E)
    if kind == "mixed":
        which = torch.randint(0, 6, (E,), generator=g)
        k[which <= 1] = torch.randint(1, 300, (E,), generator=g).int()[which <= 1]
        p[(which >= 1) & (which <= 3)] = (0.2 + 0.79 * torch.rand(E, generator=g))[(which >= 1) & (which <= 3)]
        m[which >= 3] = 0.2 * torch.rand(E, generator=g)[which >= 3]
        tau[which == 5] = 0
    return ops.Draw(cuda(tau), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p), cuda(m))


SIZES = [(1, 32768, 200, 0), (5, 1000, 60, 0), (9, 151936, 900, 0), (3, 4097, 4000, 7), (2, 31, 10, 0), (4, 1, 3, 0), (33, 5003, 17, 5), (2, 300001, 33000, 3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,V,longest,pad", SIZES)
def test_adjusted_logits(ops, E, V, longest, pad, dtype):
    g = torch.Generator().manual_seed(E + V)
    rules, l = make_rules(ops, E, V, longest, g), make_logits(E, V, dtype, g, pad)
    got = ops.adjust_logits(l, rules)
    check_adjusted(got, l, rules)
    out = torch.full((E, V + 3), 7.0, device="cuda")  # rows of another stride, off 16 bytes
    assert torch.equal(ops.adjust_logits(l, rules, out=out[:, :V]), got) and (out[:, V:] == 7).all()
    if dtype == torch.float32:
        assert torch.equal(ops.adjust_logits(l, rules, out=l), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,V,longest,pad", SIZES)
@pytest.mark.parametrize("kind", ["mixed", "free"])
def test_choice(ops, E, V, longest, pad, dtype, kind):
    g = torch.Generator().manual_seed(3 * E + V)
    rules, l, draw = make_rules(ops, E, V, longest, g), make_logits(E, V, dtype, g, pad), make_draw(ops, E, g, kind)
    tokens, logprobs = ops.choose_tokens(l, draw, rules)
    check_choice(ops.adjust_logits(l, rules), draw, tokens, logprobs)
    again = ops.choose_tokens(l, draw, rules)
    assert torch.equal(tokens, again[0]) and torch.equal(logprobs, again[1])
    tokens, logprobs = ops.choose_tokens(l, draw)  # without rules
    check_choice(l.float(), draw, tokens, logprobs)


@pytest.mark.parametrize("V", [1000, 32768, 151936])
@pytest.mark.parametrize("values", ["equal", "two", "steps", "narrow", "wide", "one", "negative"])
def test_cuts_through_equal_and_crowded_logits(ops, V, values):
    """More tokens in a bin than are put in order one by one; ties at every border go by index."""
    g = torch.Generator().manual_seed(V)
    E = 24
    l = {"equal": torch.full((E, V), 3.25), "two": torch.randint(0, 2, (E, V), generator=g).float(),
         "steps": (torch.randn(E, V, generator=g) * 8).round() / 4, "narrow": 5 + torch.rand(E, V, generator=g) * 1e-3,
         "wide": torch.randn(E, V, generator=g) * 300, "one": torch.full((E, V), -math.inf), "negative": -1e30 * torch.rand(E, V, generator=g)}[values]
    if values == "one":
        l[torch.arange(E), torch.randint(0, V, (E,), generator=g)] = -2.0
    l = l.to("cuda")
    k = torch.tensor([0, 1, 2, 7, 100, 999, V - 1, V, V + 1, 2 ** 31 - 1] * 3)[:E].to(torch.int32)
    p = torch.tensor([1.0, 0.5, 0.123, 0.999, 1.0, 0.25, 0.0] * 4)[:E]
    draw = ops.Draw(cuda(torch.full((E,), 0.9)), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)


@pytest.mark.parametrize("V", [50, 2000, 32768, 151936])
@pytest.mark.parametrize("values", ["falling", "rising", "peak", "far", "bulk"])
def test_few_and_many_likely_tokens(ops, V, values):
    """The likely ones side by side, all but one far behind the largest, or too many to be put in order at once; counts on both sides of where the
    way changes."""
    g = torch.Generator().manual_seed(7 + V)
    E = 30
    l = {"falling": torch.linspace(0, -2000, V).repeat(E, 1), "rising": torch.linspace(-300, 9, V).repeat(E, 1), "peak": torch.randn(E, V, generator=g) * 2,
         "far": torch.full((E, V), -300.0) - torch.rand(E, V, generator=g), "bulk": torch.randn(E, V, generator=g)}[values]
    if values in ("peak", "far"):
        l[:, V // 3] = 25.0
    l = l.to("cuda")
    k = torch.tensor([0, 3, 128, 383, 384, 385, 511, 512, 513, 0] * 3).to(torch.int32)
    p = torch.tensor([0.6] * 10 + [1.0] * 10 + [0.97] * 10)
    m = torch.zeros(E)
    m[9::10] = torch.tensor([1e-30, 1e-3, 0.3])
    p[19] = 1.0
    draw = ops.Draw(cuda(0.5 + torch.rand(E, generator=g)), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p), cuda(m))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)


@pytest.mark.parametrize("V", [1000, 60000])
@pytest.mark.parametrize("tau", [64.0, 1e3, 1e7, 3e38, math.inf])
def test_high_temperatures_weigh_alike_and_keep_the_order(ops, V, tau):
    g = torch.Generator().manual_seed(V)
    E = 12
    l = (torch.randn(E, V, generator=g) * 4).to("cuda")
    k = torch.tensor([0, 5, 380, 390, 900, 0, 0, 0, 700, 20, 0, 0], dtype=torch.int32)
    p = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.5, 0.001, 0.9, 0.5, 0.5, 1.0, 1.0])
    m = torch.tensor([0.0] * 10 + [0.5, 1e-6])
    draw = ops.Draw(torch.full((E,), tau, device="cuda"), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p), cuda(m))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)
    l[:, 3:-3] = -math.inf  # what is not allowed is not drawn, however high
    tokens, _ = ops.choose_tokens(l, draw)
    assert ((tokens < 3) | (tokens >= V - 3)).all()


@pytest.mark.parametrize("V", [900, 3000])
def test_order_is_the_logits_where_their_distances_from_the_largest_round_alike(ops, V):
    """Logits 1e-9 apart beside one of 8: some 480 of them are the same distance from it in 32 bits, and are ordered all the same."""
    g = torch.Generator().manual_seed(V)
    E = 64
    l = torch.stack([torch.randperm(V, generator=g) for _ in range(E)]).float() * 1e-9
    l[:, V // 2] = 8.0
    l = l.to("cuda")
    k = torch.tensor([50, 200, 390, 555, 700, 0, 0, 0] * 8).to(torch.int32)
    p = torch.tensor([1.0, 0.9, 1.0, 1.0, 0.95, 0.93, 0.8, 0.85] * 8)
    draw = ops.Draw(torch.full((E,), 1.0, device="cuda"), cuda(0.9 + 0.1 * torch.rand(E, generator=g)), cuda(k), cuda(p))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)


def test_top_k_of_equals_takes_the_first(ops):
    """Of equal logits the k first by index are kept, and u runs through them evenly."""
    V, E = 5000, 40
    l = torch.zeros(E, V, device="cuda")
    l[:, :17] = -1.0
    u = (torch.arange(E) + 0.5) / E
    draw = ops.Draw(torch.ones(E, device="cuda"), cuda(u), torch.full((E,), 20, dtype=torch.int32, device="cuda"))
    tokens, _ = ops.choose_tokens(l, draw)
    assert tokens.tolist() == [17 + int(x * 20) for x in u.tolist()]


def test_ends_of_the_uniform_numbers(ops):
    l = torch.randn(6, 3000, generator=torch.Generator().manual_seed(0)).cuda()
    l[:, 0], l[:, -1] = 1.0, 1.0
    draw = ops.Draw(torch.ones(6, device="cuda"), cuda(np.float32([0, 1 - 2.0 ** -24, 1, 7, -3, float("nan")])))
    tokens, _ = ops.choose_tokens(l, draw)
    assert tokens.tolist() == [0, 2999, 2999, 2999, 0, 0]


def test_greedy_is_the_sampler_s_choice(ops):
    from inference_engine_b200 import kernels as K

    g = torch.Generator().manual_seed(9)
    l = make_logits(12, 151936, torch.bfloat16, g)
    l[3, 500] = l[3, 100000] = 40.0
    draw = ops.Draw(torch.zeros(12, device="cuda"), torch.rand(12, generator=g).cuda())
    tokens, logprobs = ops.choose_tokens(l, draw)
    assert torch.equal(tokens, K.sample(l, 0.0, torch.zeros(1, dtype=torch.int64, device="cuda")).view(-1)) and tokens[3] == 500
    check_choice(l.float(), draw, tokens, logprobs)


def test_nothing_allowed_infinities_and_nan(ops):
    from inference_engine_b200 import kernels as K

    V = 2000
    l = torch.zeros(7, V, device="cuda")
    l[1] = -math.inf
    l[2, 5] = math.nan
    l[3] = math.nan
    l[4, 77] = l[4, 900] = math.inf
    l[5, 3:] = -math.inf
    l[6] = torch.finfo(torch.float32).min
    masks = torch.zeros(2, (V + 31) // 32, dtype=torch.int32, device="cuda")
    masks[1, 3] = 1 << 4
    for u in (0.0, 0.3, 0.9):
        rules = ops.Rules(masks=masks, mask_rows=torch.tensor([0, -1, -1, -1, -1, -1, 1], dtype=torch.int32, device="cuda"))
        draw = ops.Draw(torch.full((7,), 0.8, device="cuda"), torch.full((7,), u, device="cuda"), top_p=torch.full((7,), 0.95, device="cuda"),
                        top_k=torch.full((7,), 50, dtype=torch.int32, device="cuda"))
        K.check_status()
        tokens, logprobs = ops.choose_tokens(l, draw, rules)
        assert tokens[[0, 1, 3]].tolist() == [-1] * 3 and (logprobs[[0, 1, 3]] == -math.inf).all()
        assert 0 <= tokens[2] < 60 and tokens[2] != 5 and tokens[4] in (77, 900) and 0 <= tokens[5] < 3 and tokens[6] == 100
        assert abs(logprobs[4].item() + math.log(2)) < 1e-6 and logprobs[6] == 0
        assert K.check_status() == 0
    adj = ops.adjust_logits(l, rules)
    assert (adj[0] == -math.inf).all() and adj[2, 5].isnan() and adj[6, 100] == torch.finfo(torch.float32).min and adj[6].isinf().sum() == V - 1


def test_entries_passed_over_and_bad_numbers(ops):
    from inference_engine_b200 import kernels as K

    E, V = 6, 700
    i32 = dict(dtype=torch.int32, device="cuda")
    l = torch.randn(E, V, generator=torch.Generator().manual_seed(1)).cuda()
    history = torch.zeros(3, 5, **i32)
    history[0] = torch.tensor([4, 4, 9, 9, 9], **i32)
    pens = dict(repetition=torch.full((E,), 2.0, device="cuda"), frequency=torch.full((E,), 0.5, device="cuda"))
    draw = ops.Draw(torch.zeros(E, device="cuda"), torch.zeros(E, device="cuda"))
    K.check_status()
    rules = ops.Rules(history=history, slots=torch.tensor([-1, 0, 1, -1, 2, 0], **i32), lengths=torch.tensor([5, 5, 0, 5, 1, 3], **i32),
                      prompts=torch.tensor([0, 2, 0, 0, 1, 0], **i32), **pens)
    out = torch.full((E, V), 5.0, device="cuda")
    ops.adjust_logits(l, rules, out=out)
    assert (out[[0, 3]] == 5).all()
    check_adjusted(out, l, rules)
    tokens, logprobs = ops.choose_tokens(l, draw, rules)
    assert tokens[[0, 3]].tolist() == [-1, -1] and (tokens[[1, 2, 4, 5]] >= 0).all()
    assert K.check_status() == 0
    bad = dict(slots=[0, 3, -2, 1, 1, 1], lengths=[6, 5, 5, -1, 2, 2], mask_rows=[0, 0, 0, 0, 1, -2])
    for name, values in bad.items():
        more = {"slots": torch.zeros(E, **i32), "lengths": torch.full((E,), 2, **i32), "mask_rows": torch.zeros(E, **i32)}
        more[name] = torch.tensor(values, **i32)
        rules = ops.Rules(history=history, masks=torch.full((1, 22), -1, **i32), **more, **pens)
        out = ops.adjust_logits(l, rules)
        assert K.check_status() == 2
        tokens, _ = ops.choose_tokens(l, draw, rules)
        assert K.check_status() == 2
        assert [t >= 0 for t in tokens.tolist()] == ([True, False, False, True, True, True] if name == "slots" else [True] * E)
    history[0, 3], history[0, 4] = V, -1
    rules = ops.Rules(history=history, slots=torch.zeros(E, **i32), lengths=torch.full((E,), 5, **i32), prompts=torch.zeros(E, **i32), **pens,
                      bias_ids=torch.full((E, 1), V, **i32), bias=torch.ones(E, 1, device="cuda"))
    got = ops.adjust_logits(l, rules)
    assert K.check_status() == 2
    fine = ops.Rules(history=history, slots=torch.zeros(E, **i32), lengths=torch.full((E,), 3, **i32), prompts=torch.zeros(E, **i32), **pens)
    assert torch.equal(got, ops.adjust_logits(l, fine))


def test_tokens_are_appended(ops):
    E, V, cap = 4, 600, 9
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    history = torch.full((5, cap), -7, **i32)
    slots, lengths = torch.tensor([4, 0, -1, 2], **i32), torch.tensor([0, 8, 3, 9], **i32)
    history[0, :8] = torch.arange(8, **i32)
    history[2] = 11
    before = history.clone()
    rules = ops.Rules(history=history, slots=slots, lengths=lengths, presence=torch.ones(E, device="cuda"))
    draw = make_draw(ops, E, g, "free")
    l = make_logits(E, V, torch.bfloat16, g)
    tokens, _ = ops.choose_tokens(l, draw, rules)
    assert torch.equal(history, before)
    tokens, _ = ops.choose_tokens(l, draw, rules, append=True)
    before[4, 0], before[0, 8] = tokens[0].int(), tokens[1].int()
    assert torch.equal(history, before)  # the third is passed over, the fourth has no room


@pytest.mark.parametrize("tau", [0.0, 0.7])
def test_nothing_is_appended_behind_a_length_out_of_range(ops, tau):
    from inference_engine_b200 import kernels as K

    E, V, cap = 4, 600, 9
    i32 = dict(dtype=torch.int32, device="cuda")
    history = torch.arange(E * cap, **i32).view(E, cap)
    want = history.clone()
    rules = ops.Rules(history=history, lengths=torch.tensor([-1, cap + 1, 3, -(1 << 31)], **i32))
    draw = ops.Draw(torch.full((E,), tau, device="cuda"), torch.full((E,), 0.4, device="cuda"), torch.full((E,), 5, **i32))
    K.check_status()
    tokens, _ = ops.choose_tokens(make_logits(E, V, torch.float32, torch.Generator().manual_seed(3)), draw, rules, append=True)
    assert K.check_status() == 2
    want[2, 3] = tokens[2]
    assert torch.equal(history, want) and (tokens >= 0).all()


def test_many_biases_and_a_long_history_of_one_token(ops):
    E, V = 3, 151936
    g = torch.Generator().manual_seed(5)
    i32 = dict(dtype=torch.int32, device="cuda")
    history = torch.full((E, 70001), 1234, **i32)
    ids = torch.randint(0, 40, (E, 700), generator=g).int() * 3000
    rules = ops.Rules(history=history, lengths=torch.tensor([70001, 70000, 1], **i32), prompts=torch.tensor([1, 70000, 0], **i32),
                      frequency=torch.full((E,), 0.25, device="cuda"), repetition=torch.full((E,), 1.25, device="cuda"),
                      bias_ids=cuda(ids), bias=cuda(torch.randn(E, 700, generator=g)))
    l = make_logits(E, V, torch.float32, g)
    got = ops.adjust_logits(l, rules).double()
    want, bound = adjusted(l, rules)
    # 700 additions of a token's biases, each off by half a step of the sum so far
    per = cuda(np.stack([np.bincount(ids[e].numpy(), minlength=V) for e in range(E)])).double()
    assert ((got - cuda(want)).abs() <= cuda(bound) * (1 + per)).all()
    draw = make_draw(ops, E, g)
    tokens, logprobs = ops.choose_tokens(l, draw, rules)
    check_choice(got.float(), draw, tokens, logprobs)


def test_recorded_and_on_another_stream(ops):
    E, V = 8, 32768
    g = torch.Generator().manual_seed(6)
    rules, l, draw = make_rules(ops, E, V, 500, g), make_logits(E, V, torch.bfloat16, g), make_draw(ops, E, g)
    want = ops.choose_tokens(l, draw, rules)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.choose_tokens(l, draw, rules)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adj = ops.adjust_logits(l, rules)
        got = ops.choose_tokens(l, draw, rules)
        plain = ops.choose_tokens(adj, draw)
    for i in range(3):
        draw.uniform.copy_(torch.rand(E, generator=g))
        rules.lengths.copy_(rules.lengths.roll(1))
        l.copy_(l.roll(5, 1))
        graph.replay()
        check_adjusted(adj, l, rules)
        check_choice(adj, draw, *got)
        assert torch.equal(got[0], plain[0])


def test_empty_batch(ops):
    draw = ops.Draw(torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"))
    tokens, logprobs = ops.choose_tokens(torch.zeros(0, 100, device="cuda"), draw)
    assert tokens.shape == logprobs.shape == (0,)
    assert ops.adjust_logits(torch.zeros(0, 100, device="cuda"), ops.Rules()).shape == (0, 100)


@pytest.mark.parametrize("V", [700, 5000, 60000])
@pytest.mark.parametrize("tau", [65.0, 1e3, 5e3, 1e7, math.inf])
@pytest.mark.parametrize("values", ["ahead", "spread", "steps", "two"])
def test_cuts_at_high_temperatures_among_tokens_far_apart(ops, V, tau, values):
    """At a high temperature tokens thousands behind the largest weigh nearly as much: they count in every cut."""
    g = torch.Generator().manual_seed(V + 1)
    E = 30
    l = {"ahead": torch.randn(E, V, generator=g), "spread": torch.rand(E, V, generator=g) * 2e5, "steps": -4000.0 * torch.randint(0, 9, (E, V), generator=g),
         "two": torch.randint(0, 2, (E, V), generator=g) * 6e3}[values]
    if values == "ahead":
        l[torch.arange(E), torch.randint(0, V, (E,), generator=g)] = 1e4
    l = l.to("cuda")
    k = torch.tensor([50, 7, 383, 384, 385, 600, 2, 0, 0, 0] * 3).to(torch.int32)
    p = torch.tensor([1.0] * 7 + [0.5, 0.01, 0.97] + [0.5] * 7 + [0.999, 0.3, 0.8] + [0.9] * 10)
    m = torch.tensor([0.0] * 20 + [0.4, 1e-3] * 5)
    draw = ops.Draw(torch.full((E,), tau, device="cuda"), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p), cuda(m))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)


@pytest.mark.parametrize("V", [1500, 6000, 60000])
@pytest.mark.parametrize("tau", [0.9, 40.0, 900.0])
@pytest.mark.parametrize("values", ["different", "few", "signs"])
def test_more_logits_side_by_side_than_are_sorted_at_once(ops, V, tau, values):
    """Thousands of logits within 1e-8 of the largest keep their order, and equal ones that of their index."""
    g = torch.Generator().manual_seed(V + 2)
    E = 24
    l = {"different": torch.stack([torch.randperm(V, generator=g) for _ in range(E)]).float() * (1e-8 / V), "few": torch.randint(0, 3, (E, V), generator=g) * 1e-10,
         "signs": torch.randn(E, V, generator=g) * 1e-10}[values].to("cuda")
    k = torch.tensor([1100, 2, 37, 500, 1400, 0, 0, 0] * 3).to(torch.int32)
    p = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.5, 0.9, 0.5, 0.01] * 3)
    draw = ops.Draw(torch.full((E,), tau, device="cuda"), cuda(torch.rand(E, generator=g)), cuda(k), cuda(p))
    tokens, logprobs = ops.choose_tokens(l, draw)
    check_choice(l, draw, tokens, logprobs)


@pytest.mark.parametrize("early", [False, True])
def test_rules_and_choices_behind_one_another_see_what_was_written(ops, early):
    """Rows whose ends share lines, written over one another's, with nothing waiting in between."""
    from inference_engine_b200 import kernels as K

    E, V = 40, 20001
    g = torch.Generator().manual_seed(12)
    rules, draw = make_rules(ops, E, V, 300, g, bias=200), make_draw(ops, E, g)
    logits = [make_logits(E, V, torch.float32, g, pad=3) for _ in range(8)]
    want = []
    for l in logits:
        adj = ops.adjust_logits(l, rules)
        torch.cuda.synchronize()
        want.append((adj, *ops.choose_tokens(adj, draw)))
        torch.cuda.synchronize()
    K.set_early_start(early)
    try:
        got, over = [], torch.empty(E, V, device="cuda")
        for l in logits:
            ops.adjust_logits(l, rules, out=over)
            got.append(ops.choose_tokens(over, draw))
    finally:
        K.set_early_start(False)
    for (adj, tokens, logprobs), (t, p) in zip(want, got):
        assert torch.equal(t, tokens) and torch.equal(p, logprobs)
        check_choice(adj, draw, tokens, logprobs)
