"""What requests bring with them to a step they share, as cases that can be timed and checked.

A step of the serving loop runs one set of weights over the rows of many requests.  Three operators make room for what differs
between them:

    adapters  low-rank adapters beside the shared projections of one decoder layer: every row has its request's adapter or none
              (ops.plan_adapters once for the step's rows, ops.add_adapters for each projection)
    adjust    penalties for repeated tokens, biases and grammar masks on the logits (ops.adjust_logits)
    choose    the same and the choice of the next token with each request's own temperature, top-k, top-p and min-p
              (ops.choose_tokens); the random numbers are inputs

With `own` False the same results are computed by elementary torch operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False  # whether run() calls the framework's operators

# Shared projections of a layer as (input width, columns of each part that has a product of its own).  "A": the int8 decoder (packed query, key
# and value; output; packed gate and up; down); "B": the attention of a decoder with keys of 112 and values of 96 channels; "S": the small decoder of the tests
LAYERS = {
    "A": ((2048, (2048, 1024, 1024)), (2048, (2048,)), (2048, (6144, 6144)), (6144, (2048,))),
    "B": ((2048, (1792, 896, 768)), (1536, (2048,))),
    "S": ((256, (2048, 1024, 1024)), (2048, (256,)), (256, (512, 512)), (512, (256,))),
}
VOCABS = (1000, 32768, 151936)  # of the small decoder, of the decoders with unquantised caches, of the int8 decoder
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- the cases
def _adapters(name=None, *, rows, portions, used, rank, layer, dtype, none=0):
    """`portions` 0: decoding rows in any order; else that many prompt portions.  `none`: percent of the requests without an adapter."""
    c = {"kind": "adapters", "rows": rows, "portions": portions, "used": used, "rank": rank, "layer": layer, "dtype": dtype, "none": none}
    return c if name is None else {"name": name, **c}


def _logits(kind, name=None, *, entries, vocab, dtype, longest, mask, bias, settings="mixed"):
    """`longest`: tokens of the longest history.  `mask`: "none", "some" entries under a grammar, "empty": one of them allows nothing.  `bias`: ids per
    entry.  `settings` (choose): "greedy", "free" (a temperature and no cut), "mixed"."""
    c = {"kind": kind, "entries": entries, "vocab": vocab, "dtype": dtype, "longest": longest, "mask": mask, "bias": bias}
    if kind == "choose":
        c["settings"] = settings
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one chat turn decoding with its adapter: launches and latency
        _adapters("adapters_decode_1", rows=1, portions=0, used=1, rank=16, layer="A", dtype="bf16"),
        # a full decode batch of as many customers' adapters as fit: their weights are streamed once for a row or two each
        _adapters("adapters_decode_64", rows=64, portions=0, used=48, rank=16, layer="A", dtype="bf16", none=10),
        # a batch as traffic leaves it: odd counts, an odd rank, heads of 112 and 96 channels
        _adapters("adapters_decode_37_odd", rows=37, portions=0, used=5, rank=24, layer="B", dtype="bf16", none=30),
        # a step of long prompts: rows stream past a few adapters of high rank
        _adapters("adapters_prompt_2000", rows=2000, portions=5, used=4, rank=64, layer="A", dtype="bf16"),
        # the engine's usual prompt step at the usual rank
        _adapters("adapters_prompt_992", rows=992, portions=3, used=3, rank=16, layer="A", dtype="bf16", none=20),
        # full precision, as recorded traces are replayed
        _adapters("adapters_fp32_40", rows=40, portions=2, used=2, rank=8, layer="B", dtype="fp32"),
        # a single request with a short history and a few biases
        _logits("adjust", "adjust_1x32768", entries=1, vocab=32768, dtype="fp32", longest=200, mask="none", bias=3),
        # a full batch with long histories, half of it under a grammar
        _logits("adjust", "adjust_64x151936", entries=64, vocab=151936, dtype="bf16", longest=8192, mask="some", bias=16),
        # one request's next token: latency
        _logits("choose", "choose_1x151936", entries=1, vocab=151936, dtype="bf16", longest=300, mask="none", bias=0),
        # a full batch, every request with settings of its own
        _logits("choose", "choose_64x151936", entries=64, vocab=151936, dtype="bf16", longest=4096, mask="some", bias=8),
        # the 32-bit logits of an odd batch, one request with a grammar that allows nothing
        _logits("choose", "choose_37x32768", entries=37, vocab=32768, dtype="fp32", longest=2000, mask="empty", bias=5),
        # a batch that samples from whole distributions
        _logits("choose", "choose_64_free", entries=64, vocab=151936, dtype="bf16", longest=1024, mask="none", bias=0, settings="free"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: 1 to 2000 rows of 1 to 48 adapters of rank 8 to 64; 1 to 64 entries of the three vocabularies, or of an odd one."""
    kind = rng.choice(["adapters", "adapters", "adjust", "choose", "choose"])
    if kind == "adapters":
        dtype = "fp32" if rng.random() < 0.15 else "bf16"
        portions = rng.choice([0, 0, rng.randint(1, 6)])
        rows = _log(rng, 1, 64) if not portions else _log(rng, 8 * portions, 64 if dtype == "fp32" else 2000)
        return _adapters(rows=rows, portions=portions, used=min(_log(rng, 1, 48), rows), rank=rng.choice([8, 16, 16, 24, 32, 40, 64]),
                         layer=rng.choice("AABS") if dtype == "bf16" else rng.choice("BS"), dtype=dtype, none=rng.choice([0, 0, 20, 60]))
    vocab = rng.choice([*VOCABS, _log(rng, 500, 150000)])
    return _logits(kind, entries=_log(rng, 1, 64), vocab=vocab, dtype=rng.choice(["bf16", "fp32"]), longest=_log(rng, 4, 8192),
                   mask=rng.choice(["none", "some", "empty"]), bias=rng.choice([0, 1, 16, 100]),
                   **({"settings": rng.choice(["greedy", "free", "mixed", "mixed", "mixed"])} if kind == "choose" else {}))


# ----------------------------------------------------------------------------- adapters: inputs
def _row_adapters(case):
    """The adapter of every row, -1: none.  From the case alone, so that its work is known."""
    rng = random.Random(f"{case['rows']} {case['portions']} {case['used']} {case['none']}")
    n, used = case["rows"], case["used"]
    requests = case["portions"] or n
    of = [i if i < used else rng.randrange(used) for i in range(requests)]
    rng.shuffle(of)
    of = [-1 if rng.random() * 100 < case["none"] and of.count(a) > 1 else a for a in of]
    if not case["portions"]:
        return of
    cuts = sorted(rng.sample(range(1, n), requests - 1)) if requests > 1 else []
    return [a for a, lo, hi in zip(of, [0, *cuts], [*cuts, n]) for _ in range(hi - lo)]


def _prepare_adapters(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, R, slots, N = TYPES[case["dtype"]], case["rank"], case["used"], case["rows"]
    ids = _row_adapters(case)
    s = {"ids": torch.tensor(ids, dtype=torch.int32, device="cuda"), "slots": slots, "layers": []}
    for width, parts in LAYERS[case["layer"]]:
        def rnd(*shape, std=1.0):
            return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

        out = sum(parts)
        p = {"x": rnd(N, width), "y": rnd(N, out), "down": rnd(slots, len(parts) * R, width, std=width ** -0.5),
             "up": rnd(slots, out, R, std=0.5 * R ** -0.5), "parts": parts, "out": torch.empty(N, out, dtype=dtype, device="cuda"),
             "scale": torch.rand(slots, generator=g, device="cuda") + 0.5}
        if own:
            from inference_engine_b200 import ops

            p["adapters"] = ops.Adapters(p["down"], p["up"], p["scale"], parts)
        s["layers"].append(p)
    return s


def _run_adapters(s):
    if own:
        from inference_engine_b200 import ops

        plan = ops.plan_adapters(s["ids"], s["slots"])
        return [ops.add_adapters(p["y"], p["x"], p["adapters"], plan, out=p["out"]) for p in s["layers"]]
    # all adapters' products of every row, those of other adapters times zero
    mine = (s["ids"][:, None] == torch.arange(s["slots"], device="cuda")).float()  # [rows, slots]
    out = []
    for p in s["layers"]:
        slots, R, parts = s["slots"], p["up"].shape[2], p["parts"]
        t = (p["x"].float() @ p["down"].float().flatten(0, 1).t()).view(-1, slots, len(parts) * R) * (mine * p["scale"])[:, :, None]
        delta = [t[:, :, i * R : (i + 1) * R].flatten(1) @ up.float().transpose(1, 2).flatten(0, 1)
                 for i, up in enumerate(p["up"].split(parts, dim=1))]
        out.append((p["y"].float() + torch.cat(delta, dim=1)).to(p["y"].dtype))
    return out


def _exact_adapters(case, seed):
    s = _prepare_adapters(case, seed)
    ids, out = s["ids"].tolist(), []
    for p in s["layers"]:
        y, R = p["y"].double(), p["up"].shape[2]
        for a in sorted(set(ids) - {-1}):
            rows = torch.tensor([r for r, i in enumerate(ids) if i == a], device="cuda")
            at = 0
            for i, n in enumerate(p["parts"]):
                low = torch.einsum("rk,jk->rj", p["x"][rows].double(), p["down"][a, i * R : (i + 1) * R].double())
                y[rows, at : at + n] += p["scale"][a].double() * torch.einsum("rj,nj->rn", low, p["up"][a, at : at + n].double())
                at += n
        out.append(y)
    return out


def _work_adapters(case):
    ids, elem = _row_adapters(case), 2 if case["dtype"] == "bf16" else 4
    used, mine, R, N = len(set(ids) - {-1}), sum(i >= 0 for i in ids), case["rank"], case["rows"]
    nbytes, flops = 4 * N, 0
    for width, parts in LAYERS[case["layer"]]:
        out = sum(parts)
        nbytes += elem * (mine * width + 2 * N * out + used * R * (len(parts) * width + out))
        flops += 2 * mine * R * (len(parts) * width + out)
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------- logits: inputs
def _lengths(case):
    """(prompt, all tokens) of every entry's history."""
    rng = random.Random(f"{case['entries']} {case['longest']}")
    got = []
    for e in range(case["entries"]):
        n = case["longest"] if e == 0 else _log(rng, 1, case["longest"])
        got.append((rng.randint(1, n), n))
    return got


def _prepare_logits(case, seed):
    E, V = case["entries"], case["vocab"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    # a bulk of unlikely tokens and a few hundred that stand out, as a language model's
    logits = torch.randn(E, V, generator=g, device="cuda") * 2.0
    some = torch.randint(0, V, (E, min(300, V)), generator=g, device="cuda")
    logits.scatter_add_(1, some, uniform(*some.shape).pow(3) * 16.0)
    s = {"logits": logits.to(TYPES[case["dtype"]])}
    lengths = _lengths(case)
    # a text's tokens: few that come again and again, among them likely ones
    places = (uniform(E, case["longest"]).pow(4) * V).long().clamp_(max=V - 1)
    likely = some.gather(1, torch.randint(0, some.shape[1], places.shape, generator=g, device="cuda"))
    s["history"] = torch.where(uniform(*places.shape) < 0.3, likely, places).to(torch.int32)
    s["slots"] = torch.arange(E - 1, -1, -1, dtype=torch.int32, device="cuda")  # entries' rows of the history, in another order
    s["prompts"] = torch.tensor([a for a, _ in lengths], dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor([b for _, b in lengths], dtype=torch.int32, device="cuda")
    pick = uniform(E)
    s["repetition"] = torch.where(pick < 0.6, uniform(E, lo=1.0, hi=1.5), torch.ones(E, device="cuda"))
    s["presence"] = torch.where(pick > 0.4, uniform(E, lo=-0.5, hi=1.0), torch.zeros(E, device="cuda"))
    s["frequency"] = torch.where(pick > 0.3, uniform(E, hi=0.7), torch.zeros(E, device="cuda"))
    s["bias_ids"] = s["bias"] = s["masks"] = s["mask_rows"] = None
    if case["bias"]:
        n = case["bias"]
        s["bias_ids"] = torch.randint(0, V, (E, n), generator=g, device="cuda", dtype=torch.int32)
        s["bias_ids"][:, n - n // 3 :] = -1  # entries with fewer
        s["bias"] = uniform(E, n, lo=-8.0, hi=8.0)
    if case["mask"] != "none":
        words = (V + 31) // 32
        bits = torch.randint(-(1 << 31), 1 << 31, (4, words), generator=g, device="cuda").to(torch.int32)
        bits[0] |= torch.randint(-(1 << 31), 1 << 31, (words,), generator=g, device="cuda").to(torch.int32)  # most tokens
        bits[2] = 0  # a dozen tokens: a keyword, a bracket
        bits[2].scatter_(0, torch.randint(0, words, (12,), generator=g, device="cuda"), 1 << 7 if V > 40 else 1)
        bits[3] = 0  # nothing
        rows = [rng.choice([-1, 0, 1, 2]) for _ in range(E)]
        if case["mask"] == "empty":
            rows[rng.randrange(E)] = 3
        s["masks"], s["mask_rows"] = bits, torch.tensor(rows, dtype=torch.int32, device="cuda")
    if case["kind"] == "choose":
        kind = case["settings"]
        tau = uniform(E, lo=0.5, hi=1.4)
        k, p, m = torch.zeros(E, dtype=torch.int32), torch.ones(E), torch.zeros(E)
        for e in range(E) if kind == "mixed" else ():
            how = rng.randrange(6)
            if how in (0, 1):
                k[e] = _log(rng, 1, 200)
            if how in (1, 2, 3):
                p[e] = rng.uniform(0.5, 0.99)
            if how == 4:
                m[e] = rng.uniform(0.01, 0.2)
        greedy = uniform(E) < (1.0 if kind == "greedy" else 0.15 if kind == "mixed" else 0.0)
        s["temperature"] = torch.where(greedy, torch.zeros(E, device="cuda"), tau)
        s["top_k"], s["top_p"], s["min_p"] = k.cuda(), p.cuda(), m.cuda()
        s["uniform"] = uniform(E)
    if own:
        from inference_engine_b200 import ops

        names = ("history", "slots", "prompts", "lengths", "repetition", "presence", "frequency", "bias_ids", "bias", "masks", "mask_rows")
        s["rules"] = ops.Rules(**{n: s[n] for n in names})
        if case["kind"] == "choose":
            s["draw"] = ops.Draw(**{n: s[n] for n in ("temperature", "top_k", "top_p", "min_p", "uniform")})
    return s


# ----------------------------------------------------------------------------- logits: plain forms
def _adjusted(s):
    l = s["logits"].float()
    E, V = l.shape
    h = s["history"][s["slots"].long()].long()
    at = torch.arange(h.shape[1], device="cuda")
    seen = (at < s["lengths"][:, None]).float()
    said = seen * (at >= s["prompts"][:, None]).float()
    zero = torch.zeros(E, V, device="cuda")
    any_, out = zero.scatter_add(1, h, seen), zero.scatter_add(1, h, said)
    rep = s["repetition"][:, None]
    l = torch.where(any_ > 0, torch.where(l > 0, l / rep, l * rep), l)
    l = l - (s["frequency"][:, None] * out + s["presence"][:, None] * (out > 0).float())
    if s["bias"] is not None:
        ids = s["bias_ids"].long()
        l = l.scatter_add(1, ids.clamp(min=0), torch.where(ids >= 0, s["bias"], torch.zeros_like(s["bias"])))
    if s["masks"] is not None:
        rows = s["mask_rows"].long()
        v = torch.arange(V, device="cuda")
        allowed = (s["masks"][rows.clamp(min=0)][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        l = torch.where((allowed > 0) | (rows < 0)[:, None], l, torch.full_like(l, -math.inf))
    return l


def _chosen(s):
    l = _adjusted(s)
    E, V = l.shape
    order, index = torch.sort(l, dim=1, descending=True, stable=True)
    best = order[:, :1]
    none = best[:, 0] == -math.inf
    greedy = s["temperature"] == 0
    behind = torch.where(none[:, None], torch.zeros_like(order), best - order).double()
    w = torch.exp(-behind / torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])[:, None].double())
    rank = torch.arange(V, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    w1 = torch.where(rank < k, w, torch.zeros_like(w))
    before = w1.cumsum(1) - w1
    cut = (rank >= k) | ((before >= s["top_p"][:, None].double() * w1.sum(1, keepdim=True)) & (s["top_p"][:, None] < 1)) | (w < s["min_p"][:, None].double())
    cut[:, 0] = False
    kept = torch.zeros_like(w).scatter(1, index, torch.where(cut, torch.zeros_like(w), w))  # by token again
    sums = kept.cumsum(1)
    token = (sums <= s["uniform"][:, None].double() * sums[:, -1:]).sum(1).clamp(max=V - 1)
    token = torch.where(greedy, index[:, 0], token)
    logprob = l.double().gather(1, token[:, None])[:, 0] - torch.logsumexp(l.double(), dim=1)
    return (torch.where(none, torch.full_like(token, -1), token), torch.where(none, torch.full_like(logprob, -math.inf), logprob).float())


# ----------------------------------------------------------------------------- logits: in 64 bits from the definition
def _exact_rows(case, seed):
    import numpy as np

    s = _prepare_logits(case, seed)
    s = {k: (v.double() if v.is_floating_point() else v).cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}
    E, V = s["logits"].shape
    for e in range(E):
        l = s["logits"][e].copy()
        h = s["history"][s["slots"][e]][: s["lengths"][e]]
        out = np.bincount(h[s["prompts"][e] :], minlength=V)
        seen = np.unique(h)
        l[seen] = np.where(l[seen] > 0, l[seen] / s["repetition"][e], l[seen] * s["repetition"][e])
        l -= s["frequency"][e] * out + s["presence"][e] * (out > 0)
        for i, b in zip(s["bias_ids"][e], s["bias"][e]) if "bias" in s else ():
            if i >= 0:
                l[i] += b
        if "masks" in s and s["mask_rows"][e] >= 0:
            bits = np.unpackbits(s["masks"][s["mask_rows"][e]].view(np.uint8), bitorder="little")[:V]
            l[bits == 0] = -np.inf
        yield s, e, l


def _exact_choice(s, e, l):
    import numpy as np

    if l.max() == -np.inf:
        return -1, -np.inf
    tau, u = s["temperature"][e], s["uniform"][e]
    total = np.log(np.exp(l - l.max()).sum()) + l.max()
    order = np.argsort(-l, kind="stable")
    if tau > 0:
        if s["top_k"][e] > 0:
            order = order[: s["top_k"][e]]
        w = np.exp((l[order] - l[order[0]]) / tau)
        if s["top_p"][e] < 1:
            n = int(np.searchsorted(np.cumsum(w), s["top_p"][e] * w.sum(), side="left")) + 1
            order, w = order[:n], w[:n]
        keep = w >= s["min_p"][e]
        keep[0] = True
        order = np.sort(order[keep])
        w = np.exp((l[order] - l.max()) / tau)
        t = order[min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), len(order) - 1)]
    else:
        t = order[0]
    return int(t), float(l[t] - total)


# ----------------------------------------------------------------------------- what is called from outside
def prepare(case, seed):
    return {"kind": case["kind"], **(_prepare_adapters if case["kind"] == "adapters" else _prepare_logits)(case, seed)}


def run(state):
    if state["kind"] == "adapters":
        return _run_adapters(state)
    if not own:
        return _adjusted(state) if state["kind"] == "adjust" else _chosen(state)
    from inference_engine_b200 import ops

    if state["kind"] == "adjust":
        return ops.adjust_logits(state["logits"], state["rules"])
    return ops.choose_tokens(state["logits"], state["draw"], state["rules"])


def exact(case, seed):
    if case["kind"] == "adapters":
        return _exact_adapters(case, seed)
    import numpy as np

    if case["kind"] == "adjust":
        return np.stack([l for _, _, l in _exact_rows(case, seed)])
    got = [_exact_choice(*row) for row in _exact_rows(case, seed)]
    return np.array([t for t, _ in got], np.int64), np.array([p for _, p in got])


def work(case):
    if case["kind"] == "adapters":
        return _work_adapters(case)
    E, V, elem = case["entries"], case["vocab"], 2 if case["dtype"] == "bf16" else 4
    nbytes = E * V * elem + 4 * sum(n for _, n in _lengths(case)) + E * 60 + 8 * E * case["bias"]
    if case["mask"] != "none":
        nbytes += 4 * ((V + 31) // 32) * min(E, 4)
    if case["kind"] == "adjust":
        return {"bytes": nbytes + 4 * E * V, "flops": 4 * E * V}
    return {"bytes": nbytes + 12 * E, "flops": 8 * E * V}
