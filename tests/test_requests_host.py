"""What requests bring with them, on the host: refusals of adapters, rules and draws, of the C entry points, the scheduler's histories and a
step's fields.  No GPU."""
import ctypes

import numpy as np
import pytest
import torch

from inference_engine_b200 import _lib, ops
from inference_engine_b200.engine import PagePool, Request, Sampling, Scheduler, SlotPool, Step


def good(**kw):
    a = dict(down=torch.zeros(3, 16, 24), up=torch.zeros(3, 10, 8), scale=torch.zeros(3), parts=(6, 4))
    a.update(kw)
    return ops.Adapters(**a)


def test_adapters_as_they_are_wanted():
    a = good()
    assert (a.slots, a.rank, a.width, a.out, a.parts) == (3, 8, 24, 10, (6, 4))
    assert list(a.struct.ends)[:2] == [6, 10] and a.struct.elem == 4
    b = ops.make_adapters(2, 24, (6, 4), 3, torch.bfloat16, "cpu")
    assert b.rank == 8 and b.down.shape == (2, 16, 24)
    b.load(1, [(torch.ones(3, 24), torch.ones(6, 3)), None], 0.5)
    assert b.down[1, :3].eq(1).all() and b.down[1, 3:].eq(0).all() and b.up[1, :6, :3].eq(1).all() and b.up[1].sum() == 18 and b.scale.tolist() == [0, 0.5]
    b.clear(1)
    assert not b.down.any() and not b.up.any() and not b.scale.any()


@pytest.mark.parametrize("bad", [
    dict(parts=(6, 5)), dict(parts=()), dict(parts=(10, 0)), dict(parts=(2, 2, 2, 2, 2)), dict(scale=torch.zeros(2)), dict(scale=torch.zeros(3).double()),
    dict(up=torch.zeros(3, 10, 12), down=torch.zeros(3, 24, 24)), dict(up=torch.zeros(3, 10, 136), down=torch.zeros(3, 272, 24)), dict(down=torch.zeros(3, 8, 24)),
    dict(down=torch.zeros(3, 16, 24).bfloat16()), dict(down=torch.zeros(3, 24, 16).transpose(1, 2)), dict(up=torch.zeros(3, 80)),
    dict(down=torch.zeros(3, 16, 24).half(), up=torch.zeros(3, 10, 8).half()),
])
def test_adapters_that_are_refused(bad):
    with pytest.raises(ValueError):
        good(**bad)


@pytest.mark.parametrize("slot,pairs", [(3, [None, None]), (-1, [None, None]), (0, [None]), (0, [(torch.ones(9, 24), torch.ones(6, 9)), None]),
                                        (0, [(torch.ones(2, 23), torch.ones(6, 2)), None]), (0, [None, (torch.ones(2, 24), torch.ones(6, 2))])])
def test_weights_that_do_not_fit_a_slot(slot, pairs):
    a = good()
    with pytest.raises(ValueError):
        a.load(slot, pairs, 1.0)
    assert not a.down.any() and not a.up.any()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_rules_and_draws_as_they_are_wanted():
    r = ops.Rules(history=torch.zeros(4, 7, dtype=torch.int32), slots=ints(0, 3), lengths=ints(1, 2), masks=torch.zeros(2, 5, dtype=torch.int32),
                  mask_rows=ints(0, -1), bias_ids=torch.zeros(2, 3, dtype=torch.int32), bias=torch.zeros(2, 3))
    assert r.entries == 2 and (r.struct.capacity, r.struct.num_histories, r.struct.num_bias, r.struct.num_masks, r.struct.mask_words) == (7, 4, 3, 2, 5)
    assert ops.Rules().entries is None
    d = ops.Draw(torch.zeros(2), torch.zeros(2), top_k=ints(0, 1))
    assert d.entries == 2 and d.struct.top_k and not d.struct.top_p


@pytest.mark.parametrize("bad", [
    dict(history=torch.zeros(4, 7, dtype=torch.int32)), dict(lengths=ints(1)), dict(repetition=torch.ones(2)), dict(prompts=ints(1)),
    dict(history=torch.zeros(4, 7, dtype=torch.int64), lengths=ints(1)), dict(history=torch.zeros(7, 4, dtype=torch.int32).t(), lengths=ints(1)),
    dict(history=torch.zeros(4, 7, dtype=torch.int32), lengths=ints(1, 2), repetition=torch.ones(3)),
    dict(history=torch.zeros(4, 7, dtype=torch.int32), lengths=ints(1, 2), presence=torch.ones(2).double()),
    dict(bias=torch.zeros(2, 3)), dict(bias=torch.zeros(2, 3), bias_ids=torch.zeros(2, 4, dtype=torch.int32)), dict(bias=torch.zeros(2), bias_ids=ints(1, 2)),
    dict(masks=torch.zeros(2, 5, dtype=torch.int32)), dict(mask_rows=ints(0)), dict(masks=torch.zeros(2, 5, dtype=torch.int32), mask_rows=ints(0, 1)[::2].repeat(2)[::2]),
    dict(slots=torch.zeros(2, 2, dtype=torch.int32)),
])
def test_rules_that_are_refused(bad):
    if bad.get("mask_rows") is not None and bad.get("masks") is not None:
        bad["mask_rows"] = torch.zeros(4, dtype=torch.int32)[::2]  # not contiguous
    with pytest.raises(ValueError):
        ops.Rules(**bad)


@pytest.mark.parametrize("bad", [dict(uniform=torch.zeros(3)), dict(top_k=torch.zeros(2)), dict(top_p=torch.zeros(2).half()), dict(min_p=torch.zeros(2, 1))])
def test_draws_that_are_refused(bad):
    with pytest.raises(ValueError):
        ops.Draw(**{"temperature": torch.zeros(2), "uniform": torch.zeros(2), **bad})


def test_there_is_no_cpu_path():
    draw = ops.Draw(torch.zeros(2), torch.zeros(2))
    for call in (lambda: ops.plan_adapters(ints(0, 1), 2), lambda: ops.choose_tokens(torch.zeros(2, 5), draw), lambda: ops.adjust_logits(torch.zeros(2, 5), ops.Rules())):
        with pytest.raises(RuntimeError):
            call()


FAKE = 0x10000  # validation reads no memory


def plan(**kw):
    a = dict(order=FAKE, tiles=FAKE, max_tiles=64, tile_rows=16, num_rows=60, slots=60)
    a.update(kw)
    return _lib.AdapterPlan(*(a[n] for n, _ in _lib.AdapterPlan._fields_))


def test_adapter_entry_points_refuse():
    lib = _lib.load_decoder()
    for bad, want in [(dict(order=None), -1), (dict(tiles=FAKE + 4), -3), (dict(tile_rows=32), -2), (dict(max_tiles=62), -4), (dict(num_rows=-1), -6),
                      (dict(slots=0), -6), (dict(slots=4097), -6)]:
        assert lib.b200dec_adapter_plan(FAKE, ctypes.byref(plan(**bad)), None, None) == want, bad
    assert lib.b200dec_adapter_plan(None, ctypes.byref(plan()), None, None) == -1
    assert lib.b200dec_adapter_plan(None, ctypes.byref(plan(num_rows=0)), None, None) == 0

    def add(ad=None, pl=None, **kw):
        a = dict(down=FAKE, up=FAKE, scale=FAKE, slots=60, rank=16, width=64, parts=2, elem=2)
        a.update(ad or {})
        st = _lib.Adapters(*(a[n] for n, _ in _lib.Adapters._fields_[:-1]))
        st.ends[:4] = a.get("ends", [32, 48, 0, 0])
        v = dict(x=FAKE, xs=64, y=2 * FAKE, ys=48, out=3 * FAKE, os=48, ws=None, n=0)
        v.update(kw)
        return lib.b200dec_add_adapters(ctypes.byref(st), ctypes.byref(plan(**(pl or {}))), v["x"], v["xs"], v["y"], v["ys"], v["out"], v["os"], v["ws"], v["n"],
                                        None, None)

    assert add(ad=dict(down=None)) == add(x=None) == add(out=None) == -1
    for ad in (dict(slots=59), dict(rank=12), dict(rank=136), dict(rank=0), dict(parts=0), dict(parts=5), dict(elem=1), dict(width=0), dict(ends=[32, 32, 0, 0]),
               dict(ends=[0, 32, 0, 0])):
        assert add(ad=ad) == -2, ad
    assert add(xs=63) == add(ys=47) == add(os=47) == add(out=FAKE) == add(out=2 * FAKE, os=56) == -2
    assert add(ad=dict(down=FAKE + 8)) == add(y=2 * FAKE + 1) == -3
    many = dict(num_rows=600, tile_rows=128, max_tiles=65)
    high = dict(rank=64)  # (whole tiles)
    assert add(high, many) == -4 and add(high, many, ws=FAKE, n=100) == -4 and add(high, many, ws=FAKE + 8, n=1 << 30) == -3
    st = _lib.Adapters(FAKE, FAKE, FAKE, 60, 24, 64, 2, 2)
    assert lib.b200dec_add_adapters_workspace(ctypes.byref(st), ctypes.byref(plan(**many))) == 65 * 2 * 16384
    assert lib.b200dec_add_adapters_workspace(ctypes.byref(st), ctypes.byref(plan())) == 0


def test_logit_entry_points_refuse():
    lib = _lib.load_decoder()

    def rules(**kw):
        a = {n: None for n, _ in _lib.Rules._fields_}
        a.update(capacity=0, num_histories=0, num_bias=0, num_masks=0, mask_words=0)
        a.update(kw)
        return _lib.Rules(*(a[n] for n, _ in _lib.Rules._fields_))

    def adjust(r=None, logits=FAKE, stride=100, elem=2, out=2 * FAKE, os=100, E=3, V=100):
        return lib.b200dec_adjust_logits(logits, stride, elem, ctypes.byref(r or rules()), out, os, E, V, None, None)

    def choose(r=None, logits=FAKE, stride=100, elem=2, E=3, V=100, **draw):
        d = dict(temperature=FAKE, top_k=None, top_p=None, min_p=None, uniform=FAKE)
        d.update(draw)
        return lib.b200dec_choose_tokens(logits, stride, elem, ctypes.byref(r or rules()), ctypes.byref(_lib.Draw(*(d[n] for n, _ in _lib.Draw._fields_))), E, V, 0,
                                         FAKE, FAKE, None, None)

    assert adjust(E=0) == choose(E=0) == 0
    assert adjust(logits=None) == adjust(out=None) == choose(logits=None) == choose(uniform=None) == -1
    assert adjust(stride=99) == adjust(os=99) == adjust(elem=1) == adjust(out=FAKE) == choose(stride=99) == choose(elem=8) == -2
    assert adjust(V=0) == adjust(E=65536) == choose(V=0) == choose(V=393217, stride=400000) == choose(E=-1) == -6
    assert adjust(logits=FAKE + 1) == adjust(out=2 * FAKE + 2) == choose(logits=FAKE + 1) == choose(top_p=FAKE + 2) == -3
    for call in (adjust, choose):
        assert call(rules(history=FAKE)) == call(rules(num_bias=2, bias=FAKE)) == call(rules(masks=FAKE, num_masks=1, mask_words=4)) == -1
        assert call(rules(history=FAKE, lengths=FAKE)) == call(rules(masks=FAKE, mask_rows=FAKE, num_masks=1, mask_words=3)) == -2
        assert call(rules(history=FAKE, lengths=FAKE, capacity=-1)) == -6
        assert call(rules(presence=FAKE + 1)) == -3


@pytest.mark.parametrize("bad", [dict(temperature=-0.1), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=1.5), dict(repetition=0.0),
                                 dict(presence=float("nan")), dict(bias={3: float("inf")}), dict(bias={3: 1e300}), dict(temperature=3.5e38),
                                 dict(top_k=2 ** 31), dict(repetition=1e-60), dict(seed=-1)])
def test_sampling_that_is_refused(bad):
    with pytest.raises(ValueError):
        Sampling(**bad)


def make_scheduler(histories):
    return Scheduler(2, 64, 16, PagePool(64), 24, 8, -1, None, SlotPool(histories))


def test_histories_are_handed_out_and_come_back():
    s = make_scheduler(2)
    a, b, c = (s.submit([1, 2, 3], 4) for _ in range(3))
    st = s.plan()
    assert (a.history, b.history, c.history) == (0, 1, -1)
    s.commit(st, [5, -1])  # nothing is allowed for the second one: it ends without a token
    assert a.output == [5] and b.output == [] and b.t_finish is not None and b.t_first_token is None and b.history == -1 and b.pages == []
    st = s.plan()
    assert c.history == 1 and [r.id for r, _ in st.entries] == [a.id, c.id]
    s = Scheduler(2, 64, 16, PagePool(64), 24, 8, -1)  # without histories a token is a token
    r = s.submit([1], 4)
    s.commit(s.plan(), [-1])
    assert r.output == [-1] and r.history == -1


def test_a_step_s_fields():
    """Engine.fill_asks and asks_views, without a device."""
    from inference_engine_b200.engine import Engine

    class Fake(Engine):
        def __init__(self):
            self.np, self.torch = np, torch
            self.own_sampling, self.max_bias, self.adapter_slots = True, 2, 3
            self.history = torch.zeros(4, 16, dtype=torch.int32)
            self.masks = torch.zeros(2, 1, dtype=torch.int32)

    eng = Fake()
    rng = type("R", (), {"random": lambda self: 0.25})()
    mk = lambda i, prompt, **kw: Request(i, prompt, 5, rng=rng, **kw)  # noqa: E731
    first = mk(0, [7, 8], history=2, output=[9], cached_len=2, adapter=1,
               sampling=Sampling(temperature=0.5, top_k=3, top_p=0.75, bias={4: -1.5}, grammar=lambda out: len(out)))
    part = mk(1, [1, 2, 3, 4, 5], history=0, cached_len=1, adapter=0)  # in the middle of its prompt
    replayed = mk(2, [], adapter=2)
    step = Step([(first, [9]), (part, [2, 3]), (replayed, [6])], 1)
    n = eng.asks_size(6, 8)
    buf = np.full(n, 77, np.int32)
    eng.fill_asks(buf, step, 6, 8)
    asks = eng.asks_views(torch.from_numpy(buf), 6, 8)["asks"]
    assert asks.adapters.tolist() == [1, 0, 0, 2, -1, -1, -1, -1]
    r, d = asks.rules, asks.draw
    assert r.slots.tolist() == [2, -1, -1, -1, -1, -1] and r.lengths.tolist() == [3, 0, 0, 0, 0, 0] and r.prompts.tolist()[0] == 2
    assert r.mask_rows.tolist() == [1, -1, -1, -1, -1, -1] and r.bias_ids.tolist()[0] == [4, -1] and r.bias[0, 0] == -1.5 and (r.bias_ids[1:] == -1).all()
    assert d.temperature.tolist() == [0.5, 0, 0, 0, 0, 0] and d.top_k.tolist()[0] == 3 and d.top_p.tolist() == [0.75] + [1] * 5 and d.uniform[0] == 0.25
    assert r.repetition.tolist() == [1] * 6
    few = eng.asks_views(torch.from_numpy(buf), 6, 8, 2, 3)["asks"]
    assert few.adapters.tolist() == [1, 0, 0] and few.rules.slots.tolist() == [2, -1] and few.rules.bias.shape == (2, 2)
    eng.own_sampling, eng.adapter_slots = False, 0
    assert eng.asks_size(6, 8) == 0 and eng.asks_views(torch.zeros(0, dtype=torch.int32), 6, 8) == {}
    first = mk(0, [7, 8], history=2, output=[9, 9, 9], cached_len=4, sampling=Sampling(grammar=lambda out: 2))
    eng.own_sampling = True
    with pytest.raises(ValueError):
        eng.fill_asks(np.zeros(eng.asks_size(6, 8), np.int32), Step([(first, [9])], 1), 6, 8)


def host_engine(max_batch=3):
    """An engine whose steps run on the host: a request's next token is its random number in thousandths."""
    from types import SimpleNamespace

    from inference_engine_b200.engine import Engine

    class OnHost(Engine):
        def __init__(self):
            self.np, self.torch, self.model, self.tau = np, torch, SimpleNamespace(vocab=1000), 0.0
            self.own_sampling, self.max_bias, self.adapter_slots, self.seed = True, 2, 0, 9
            self.history, self.masks = torch.zeros(max_batch, 64, dtype=torch.int32), torch.full((2, 32), -1, dtype=torch.int32)
            self.pool = PagePool(64)
            self.sched = Scheduler(max_batch, 64, 16, self.pool, 24, 8, -1, None, SlotPool(max_batch))
            self.rows, self.steps, self.seconds = {}, [], {"plan": 0.0, "run (inputs, launch, read-back)": 0.0, "commit": 0.0}

        def run(self, step):
            assert step.entries and [r.decoding for r, _ in step.entries] == [i < step.num_decoding for i in range(len(step.entries))]
            self.steps.append([r.id for r, _ in step.entries])
            n = len(step.entries)
            buf = np.zeros(self.asks_size(n, 8), np.int32)
            self.fill_asks(buf, step, n, 8)
            return SimpleNamespace(tokens=(self.asks_views(torch.from_numpy(buf), n, 8)["asks"].draw.uniform * 1000).long())

    return OnHost()


@pytest.mark.parametrize("when,how", [(0, "raise"), (2, "raise"), (0, "row"), (3, "row")])
def test_a_grammar_that_fails_ends_its_own_request(monkeypatch, when, how):
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)

    def grammar(out):
        if len(out) == when:
            if how == "raise":
                raise KeyError("no such state")
            return 2
        return len(out) % 2

    prompts, sampling = [[1, 2], [3] * 20, [4], [5, 6, 7]], Sampling(temperature=1.0)
    alone = []
    for i, p in enumerate(prompts):
        eng = host_engine()
        eng.sched.next_id = i
        alone.append(eng.generate([p], 6, sampling)[0].output)
    eng = host_engine()
    for p in prompts:
        eng.submit_request(p, 6, sampling)
    bad = eng.sched.waiting[2]
    bad.sampling = Sampling(temperature=1.0, grammar=grammar)
    reqs, ended = list(eng.sched.waiting), []
    for _ in range(40):
        ended += eng.step()
    assert eng.sched.idle() and sorted(r.id for r in ended) == [0, 1, 2, 3]
    assert isinstance(bad.error, KeyError if how == "raise" else ValueError) and bad.t_finish is not None
    assert [r.output for r in reqs] == [a[:when] if i == 2 else a for i, a in enumerate(alone)]
    assert all(r.error is None for r in reqs if r is not bad)
    assert eng.pool.uncommitted() == eng.pool.capacity and eng.sched.histories.free == [2, 1, 0] and not eng.rows


def test_a_failed_request_keeps_no_engine_alive():
    import gc
    import weakref

    def grammar(out):
        try:
            raise KeyError("first")
        except KeyError:
            raise LookupError("then")

    eng = host_engine()
    r = eng.submit_request([1], 3, Sampling(grammar=grammar))
    alive = weakref.ref(eng)
    gc.disable()
    try:
        assert eng.step() == [r]
        del eng
        assert alive() is None
    finally:
        gc.enable()
    assert isinstance(r.error, LookupError) and "in grammar" in r.error.__notes__[0] and "first" in r.error.__notes__[0]


def test_a_step_of_requests_that_all_fail(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    eng = host_engine()
    reqs = [eng.submit_request([1], 3, Sampling(grammar=lambda out: 7)) for _ in range(4)]
    assert {r.id for r in eng.step()} == {0, 1, 2} and eng.steps == [] and eng.step() == [reqs[3]] and eng.step() == [] and eng.sched.idle()
    calls = []
    r = eng.submit_request([1, 2, 3], 4, Sampling(grammar=lambda out: calls.append(list(out)) or 0))
    while not eng.sched.idle():
        eng.step()
    assert len(r.output) == 4 and calls == [r.output[:n] for n in range(4)]  # once for each token


def test_requests_without_a_way_of_sampling_have_the_engine_s_temperature():
    eng = host_engine()
    assert eng.submit_request([1], 2).sampling is None
    eng.tau = 0.75
    r, own = eng.submit_request([1], 2), eng.submit_request([1], 2, Sampling())
    assert r.sampling == Sampling(0.75) and own.sampling.temperature == 0
    eng.own_sampling = False  # the sampler that all requests share
    assert eng.submit_request([1], 2).sampling is None


def test_early_starts_can_be_switched_off():
    """In a process of its own: what is said before a library is loaded holds for it too."""
    import subprocess
    import sys

    code = """
from inference_engine_b200 import _lib, kernels as K
lib = _lib.load()
both = lambda: (lib.b200kv_get_chained_launch(), lib.b200kv_get_early_launch())
assert both() == (0, 1)
K.set_early_start(False)
dec = _lib.load_decoder()
assert both() == (0, 0) and (dec.b200kv_get_chained_launch(), dec.b200kv_get_early_launch()) == (0, 0)
K.set_early_start(True)
assert both() == (1, 1) and (dec.b200kv_get_chained_launch(), dec.b200kv_get_early_launch()) == (1, 1)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
