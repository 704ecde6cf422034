"""What requests bring with them, through the engine: their adapters, their ways of sampling, their grammars, recorded and not."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import biranex_helpers, radivik_helpers as H
from tests.test_gpu_token_choice import check_choice

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def scaffold(vocab=1000):
    from inference_engine_b200 import scaffold as S

    return S.DecoderScaffold(torch.device("cuda", 0), hidden=256, ffn=512, vocab=vocab, layers=2, seed=7)


def build(model, use_graphs, **kw):
    from inference_engine_b200.engine import Engine

    args = dict(max_batch_size=4, max_len=512, stop_token_id=-1, max_tokens_per_step=96, min_first_chunk=16, max_graph_tokens=96, use_graphs=use_graphs)
    args.update(kw)
    return Engine(model, **args)


def prompts():
    g = torch.Generator().manual_seed(3)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 150, 33, 70, 16, 201)]


def status_clear():
    from inference_engine_b200 import kernels as K

    assert K.check_status() == 0


def fill(model, slot, seed, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for layer in model.adapters:
        for ad in layer.values():
            r = 6 if seed % 2 else 8
            ad.load(slot, [(torch.randn(r, ad.width, generator=g, device="cuda") * ad.width ** -0.5, torch.randn(n, r, generator=g, device="cuda") * gain * r ** -0.5)
                           for n in ad.parts], 0.5)


@pytest.mark.parametrize("use_graphs", [False, True])
def test_requests_that_ask_nothing_get_what_they_got(use_graphs):
    plain = [r.output for r in build(scaffold(), use_graphs).generate(prompts(), 6)]
    model = scaffold()
    model.make_adapters(3, 8)
    fill(model, 1, 5)
    eng = build(model, use_graphs, own_sampling=True, adapters=True)
    assert [r.output for r in eng.generate(prompts(), 6)] == plain
    assert [r.output for r in eng.generate(prompts(), 6, adapter=2)] == plain  # an empty slot
    assert eng.sched.histories.free == [3, 2, 1, 0] and eng.sched.idle() and eng.pool.committed == 0
    status_clear()


def test_adapters_recorded_and_not_and_in_other_slots():
    outs = []
    for use_graphs, slots in ((False, (0, 1, 2)), (True, (0, 1, 2)), (True, (4, 2, 0))):
        model = scaffold()
        model.make_adapters(5, 8)
        for i, s in enumerate(slots):
            fill(model, s, 10 + i)
        eng = build(model, use_graphs, adapters=True)
        reqs = [eng.submit_request(p, 6, adapter=-1 if i % 4 == 3 else slots[i % 4]) for i, p in enumerate(prompts())]
        while not eng.sched.idle():
            eng.step()
        outs.append([r.output for r in reqs])
        status_clear()
    assert outs[0] == outs[1] == outs[2]
    assert outs[0] != [r.output for r in build(scaffold(), True).generate(prompts(), 6)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("graphs", [False, True])
def test_an_adapter_is_the_sum_of_weights(dtype, graphs):
    """Logits of requests with adapters against the plain implementation on weights that hold the products."""
    cfg = H.small()
    w = H.weights(cfg, 1)
    m = H.model(cfg, w, dtype)
    m.make_adapters(3, 8)
    merged = [dict(w), dict(w), dict(w)]
    for slot in (0, 2):
        g = np.random.default_rng(slot)
        for i, (layer, own) in enumerate(zip(cfg["layers"], m.adapters)):
            p = f"l{i}.mix."
            for name, keys in (("qkv", ["q", "k", "v"][: len(own["qkv"].parts)]), ("o", ["o"])):
                ad, pairs = own[name], []
                for key, n in zip(keys, ad.parts):
                    d, u = (H.bf16(g.standard_normal(s) * s[1] ** -0.5) for s in ((5, ad.width), (n, 5)))
                    pairs.append((torch.tensor(d), torch.tensor(u)))
                    merged[slot][p + key] = (w[p + key] + 0.375 * (u.astype(np.float64) @ d)).astype(np.float32)
                ad.load(slot, pairs, 0.375)
    eng = H.engine(m, graphs=graphs, adapters=True)
    rng = np.random.default_rng(3)
    tokens = [rng.integers(0, cfg["vocab"], n).tolist() for n in (70, 33, 41)]
    tokens = [H.settle(cfg, merged[s], t) for s, t in zip((0, 2, 1), tokens)]  # the last slot is empty
    live = [eng.open_replay() for _ in tokens]
    for r, s in zip(live, (0, 2, -1)):
        r.adapter = s
    got, at = [[], [], []], [0, 0, 0]
    for plan in ([40, 3, 0], [1, 1, 20], [29, 1, 1], [0, 28, 20]):  # portions beside decoding rows
        entries = [(live[i], tokens[i][at[i] : at[i] + n], list(range(n))) for i, n in enumerate(plan) if n]
        logits, o = eng.replay(entries).numpy(), 0
        for i, n in enumerate(plan):
            got[i].append(logits[o : o + n])
            o += n
            at[i] += n
    for i, slot in enumerate((0, 2, 1)):
        assert H.error(np.concatenate(got[i]), H.oracle_logits(cfg, merged[slot], tokens[i])).max() < H.TOLERANCE[dtype], i
    status_clear()


def test_tokens_are_drawn_as_each_request_asks():
    """Every step's logits are kept; the tokens follow from them, the histories and the requests' own random numbers."""
    from inference_engine_b200 import ops
    from inference_engine_b200.engine import Sampling

    allowed = {0: [3, 17, 500, 999], 1: list(range(0, 1000, 3))}
    asks = [Sampling(temperature=0.9, top_k=7, seed=5), Sampling(temperature=1.3, top_p=0.8, repetition=1.4, presence=0.3, frequency=0.2),
            Sampling(bias={1: 4.0, 20: -9.0, 999: 2.5}, frequency=0.5), Sampling(temperature=0.8, min_p=0.1, grammar=lambda out: len(out) % 2),
            None, Sampling(temperature=1.0, grammar=lambda out: 0 if len(out) < 3 else -1, repetition=2.0)]
    outs = []
    for use_graphs in (False, True):
        model = scaffold()
        eng = build(model, use_graphs, own_sampling=True, seed=21)
        for row, ids in allowed.items():
            eng.set_mask(row, ids)
        reqs = [eng.submit_request(p, 7, s) for p, s in zip(prompts(), asks)]
        seen, logits = {r.id: [] for r in reqs}, []
        if not use_graphs:
            inner = model.logits
            model.logits = lambda h: logits.append(inner(h)) or logits[-1]
        while not eng.sched.idle():
            before = {r.id: len(r.output) for r in reqs}
            plan, step = eng.sched.plan, []
            eng.sched.plan = lambda: step.append(plan()) or step[-1]
            eng.step()
            eng.sched.plan = plan
            if not use_graphs:
                for row, (r, _) in enumerate(step[0].entries):
                    if len(r.output) > before[r.id]:
                        seen[r.id].append(logits[-1][row].float().cpu())
        assert all(len(r.output) == 7 for r in reqs) and eng.sched.histories.free == [3, 2, 1, 0]
        outs.append([r.output for r in reqs])
        status_clear()
        if use_graphs:
            continue
        for r, s in zip(reqs, asks):
            s = s or Sampling()
            rng = np.random.default_rng([21, r.id] if s.seed is None else s.seed)
            l = torch.stack(seen[r.id]).cuda()
            n = len(l)
            i32 = dict(dtype=torch.int32, device="cuda")
            hist = torch.tensor(r.prompt_ids + r.output, **i32)[None]
            masks = torch.full((3, 32), -1, **i32)
            masks[:2] = eng.masks[:2]
            rows = [-1 if s.grammar is None else s.grammar(r.output[:j]) for j in range(n)]
            rules = ops.Rules(history=hist, slots=torch.zeros(n, **i32), lengths=torch.arange(len(r.prompt_ids), len(r.prompt_ids) + n, **i32),
                              prompts=torch.full((n,), len(r.prompt_ids), **i32), repetition=torch.full((n,), s.repetition, device="cuda"),
                              presence=torch.full((n,), s.presence, device="cuda"), frequency=torch.full((n,), s.frequency, device="cuda"),
                              bias_ids=torch.tensor([list(s.bias) or [-1]] * n, **i32), bias=torch.tensor([list(s.bias.values()) or [0.0]] * n, device="cuda"),
                              masks=masks, mask_rows=torch.tensor(rows, **i32))
            adj = ops.adjust_logits(l, rules)
            full = lambda x, t=torch.float32: torch.full((n,), x, dtype=t, device="cuda")  # noqa: E731
            draw = ops.Draw(full(s.temperature), torch.tensor([rng.random() for _ in range(n)], dtype=torch.float32, device="cuda"),
                            full(s.top_k, torch.int32), full(s.top_p), full(s.min_p))
            logprobs = torch.log_softmax(adj.double(), 1).gather(1, torch.tensor(r.output, device="cuda")[:, None])[:, 0]
            check_choice(adj, draw, torch.tensor(r.output), logprobs)
            for j, row in enumerate(rows):
                assert row < 0 or r.output[j] in allowed[row]
    assert outs[0] == outs[1]


def test_a_request_s_random_numbers_are_its_own():
    from inference_engine_b200.engine import Sampling

    s = [Sampling(temperature=1.0, seed=i) for i in range(4)]
    alone = []
    for i in range(4):
        eng = build(scaffold(), True, own_sampling=True)
        alone.append(eng.generate([[1, 2, 3]], 5, s[i])[0].output)
    assert len({tuple(a) for a in alone}) > 1
    a, b = (build(scaffold(), True, own_sampling=True, seed=n).generate([[1, 2, 3], [1, 2, 3]], 5, Sampling(temperature=1.0)) for n in (1, 2))
    assert a[0].output != a[1].output and a[0].output != b[0].output
    again = build(scaffold(), True, own_sampling=True, seed=1).generate([[1, 2, 3], [1, 2, 3]], 5, Sampling(temperature=1.0))
    assert [r.output for r in again] == [r.output for r in a]


@pytest.mark.parametrize("use_graphs", [False, True])
def test_a_grammar_that_allows_nothing_ends_its_request(use_graphs):
    from inference_engine_b200.engine import Sampling

    eng = build(scaffold(), use_graphs, own_sampling=True)
    eng.set_mask(0, [])
    eng.set_mask(1, [42])
    p = prompts()
    a = eng.submit_request(p[0], 6, Sampling(grammar=lambda out: 1 if len(out) < 2 else 0))
    b = eng.submit_request(p[2], 6)
    c = eng.submit_request(p[3], 6, Sampling(temperature=1.0, grammar=lambda out: 0))
    while not eng.sched.idle():
        eng.step()
    assert a.output == [42, 42] and c.output == [] and len(b.output) == 6 and all(r.t_finish is not None for r in (a, b, c))
    assert eng.pool.uncommitted() == eng.pool.capacity and eng.sched.histories.free == [3, 2, 1, 0]
    status_clear()


def test_what_is_refused():
    from inference_engine_b200.engine import Sampling

    model = scaffold()
    with pytest.raises(ValueError):
        build(model, False, adapters=True)
    eng = build(model, False)
    with pytest.raises(ValueError):
        eng.submit_request([1], 2, Sampling())
    with pytest.raises(ValueError):
        eng.submit_request([1], 2, adapter=0)
    with pytest.raises(ValueError):
        eng.set_mask(0, [1])
    model.make_adapters(2, 8)
    eng = build(model, False, adapters=True, own_sampling=True, max_bias=1, num_masks=2)
    for kw in (dict(adapter=2), dict(adapter=-2), dict(sampling=Sampling(bias={1: 1.0, 2: 1.0})), dict(sampling=Sampling(bias={1000: 1.0}))):
        with pytest.raises(ValueError):
            eng.submit_request([1], 2, **kw)
    with pytest.raises(ValueError):
        eng.submit_request([1, 1000], 2)
    for row, ids in ((2, [1]), (-1, [1]), (0, [1000]), (0, [-1])):
        with pytest.raises(ValueError):
            eng.set_mask(row, ids)
    assert eng.sched.idle()
    eng = build(model, False, own_sampling=True, seed=-3)  # (any number is a seed of an engine)
    assert len(eng.generate([[1, 2]], 2, Sampling(temperature=1.0))[0].output) == 2


@pytest.mark.parametrize("graphs", [False, True])
def test_a_model_with_states(graphs):
    """Biranex takes ways of sampling; requests that ask nothing get what they got, replay is what it was."""
    from inference_engine_b200.engine import Sampling

    B = biranex_helpers
    cfg = B.CONFIGS["small"]
    model = B.model(cfg, B.weights(cfg, 1), torch.float32)
    args = dict(graphs=graphs)
    p = [np.random.default_rng(n).integers(0, cfg["vocab"], n).tolist() for n in (9, 30, 17)]
    plain = [r.output for r in B.engine(model, **args).generate(p, 5)]
    eng = B.engine(model, own_sampling=True, **args)
    assert [r.output for r in eng.generate(p, 5)] == plain
    some = eng.generate(p, 5, Sampling(temperature=1.5, top_p=0.95, repetition=1.2))
    assert all(len(r.output) == 5 for r in some)
    with pytest.raises(ValueError):
        B.engine(model, adapters=True, **args)
    status_clear()


def test_command_line(tmp_path):
    cfg = dict(architecture="DecoderScaffold", hidden=256, ffn=512, vocab=1000, layers=1)
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    base = [sys.executable, "-m", "inference_engine_b200", "generate", "--model", str(tmp_path), "--random-weights", "--prompt", "5 6 7", "--max-new-tokens", "4"]

    def run(*more):
        out = subprocess.run(base + list(more), cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr[-2000:]
        return json.loads(out.stdout.splitlines()[-1])["output"]

    greedy = run()
    assert run("--top-k", "1", "--tau", "1.0") == greedy
    assert len(run("--tau", "0.9", "--top-p", "0.9", "--repetition-penalty", "1.3", "--frequency-penalty", "0.1", "--presence-penalty", "0.1", "--min-p", "0.01")) == 4


@pytest.mark.parametrize("use_graphs", [False, True])
def test_a_grammar_that_fails_ends_its_request_and_no_other(use_graphs):
    from inference_engine_b200.engine import Sampling

    def outputs(grammar):
        eng = build(scaffold(), use_graphs, own_sampling=True, seed=4)
        reqs = [eng.submit_request(p, 6, Sampling(temperature=1.0, top_k=9, grammar=grammar if i == 1 else None)) for i, p in enumerate(prompts()[:4])]
        while not eng.sched.idle():
            eng.step()
        assert eng.pool.uncommitted() == eng.pool.capacity and eng.sched.histories.free == [3, 2, 1, 0]
        return reqs

    def failing(out):
        return -1 if len(out) < 2 else 1 // 0

    whole, cut = outputs(lambda out: -1), outputs(failing)
    assert isinstance(cut[1].error, ZeroDivisionError) and cut[1].output == whole[1].output[:2]
    assert [r.output for i, r in enumerate(cut) if i != 1] == [r.output for i, r in enumerate(whole) if i != 1]
    status_clear()


@pytest.mark.parametrize("use_graphs", [False, True])
def test_the_engine_s_temperature_is_that_of_requests_without_their_own(use_graphs):
    from inference_engine_b200.engine import Sampling

    def outputs(sampling, **kw):
        return [r.output for r in build(scaffold(), use_graphs, own_sampling=True, seed=2, **kw).generate(prompts()[:3], 6, sampling)]

    assert outputs(None, tau=1.5) == outputs(Sampling(1.5)) != outputs(None) == outputs(Sampling(), tau=1.5)


@pytest.mark.parametrize("use_graphs", [False, True])
def test_slots_made_anew_behind_the_engine_s_back_are_refused(use_graphs):
    """Recorded steps would read memory that the old slots had."""
    model = scaffold()
    model.make_adapters(3, 8)
    eng = build(model, use_graphs, adapters=True)
    fill(model, 1, 5)
    want = eng.generate([[1, 2, 3]], 3, adapter=1)[0].output
    old = model.adapters
    model.make_adapters(1, 8)
    eng.submit_request([1, 2, 3], 3, adapter=1)
    with pytest.raises(RuntimeError, match="slots"):
        eng.step()
    model.adapters = old
    r, = eng.sched.running
    while not eng.sched.idle():
        eng.step()
    assert r.output == want
    status_clear()


def test_adapters_and_ways_of_sampling_in_the_same_steps():
    """Every request with an adapter, a grammar or a way of sampling, or several of them: tokens follow from the step's logits, which follow from the adapters."""
    from inference_engine_b200 import ops
    from inference_engine_b200.engine import Sampling

    even = list(range(0, 1000, 2))
    asks = [(0, Sampling(temperature=0.9, top_k=12, seed=1)), (2, Sampling(temperature=1.1, top_p=0.9, frequency=0.4, grammar=lambda out: len(out) % 2 - 1)),
            (-1, Sampling(repetition=1.3, bias={7: 3.0})), (2, None), (1, Sampling(temperature=0.7, min_p=0.05, grammar=lambda out: 0)), (-1, None)]

    def run(use_graphs, adapters=True, watch=None):
        model = scaffold()
        model.make_adapters(3, 8)
        for slot in range(3):
            fill(model, slot, 20 + slot)
        eng = build(model, use_graphs, adapters=True, own_sampling=True, seed=13)
        eng.set_mask(0, even)
        reqs = [eng.submit_request(p, 6, s, adapter=a if adapters else -1) for p, (a, s) in zip(prompts(), asks)]
        if watch is not None:
            choose = ops.choose_tokens
            watch.append((choose, []))

            def keep(logits, draw, rules, append):
                l, same = logits.clone(), lambda t: None if t is None else t.clone()  # noqa: E731
                own = ops.Draw(*(same(getattr(draw, n)) for n in ("temperature", "uniform", "top_k", "top_p", "min_p")))
                r = ops.Rules(**{k: same(v) for k, v in vars(rules).items() if k in ops.Rules.__dataclass_fields__})
                got = choose(logits, draw, rules, append)
                watch[0][1].append((l, own, r, got))
                return got

            ops.choose_tokens = keep
        try:
            while not eng.sched.idle():
                eng.step()
        finally:
            if watch is not None:
                ops.choose_tokens = watch[0][0]
        status_clear()
        return [r.output for r in reqs]

    seen = []
    eager = run(False, watch=seen)
    assert eager == run(True) and all(len(o) == 6 for o in eager)
    assert all(t % 2 == 0 for t in eager[4]) and all(t % 2 == 0 for t in eager[1][1::2])
    without = run(False, adapters=False)
    assert all((a == b) == (ask[0] < 0) for a, b, ask in zip(eager, without, asks))
    for l, draw, rules, (tokens, logprobs) in seen[0][1]:
        live = rules.slots >= 0
        assert ((tokens >= 0) == live).all()
        adj = ops.adjust_logits(l, rules, out=torch.full(l.shape, -float("inf"), device="cuda"))  # (rows that are passed over: nothing)
        check_choice(adj, draw, tokens, logprobs)
