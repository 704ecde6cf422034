"""Low-rank adapters of many requests beside a shared projection, against the formula in 64 bits.

Bound per element: both sums in 32 bits over `width` and `rank` terms (each addition and product off by at most a step, 2^-23 of the
sum of magnitudes), in bf16 the inner values as two terms (2^-16 of each), the result rounded once (half a step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from inference_engine_b200 import ops

    return ops


def make(ops, rows, width, parts, rank, slots, dtype, seed=0, ids=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    ad = ops.Adapters(rnd(slots, len(parts) * rank, width, std=width ** -0.5), rnd(slots, sum(parts), rank, std=0.5),
                      torch.rand(slots, generator=g, device="cuda") + 0.5, parts)
    if ids is None:
        ids = torch.randint(-1, slots, (rows,), generator=g, device="cuda")
    return ad, ids.to("cuda", torch.int32), rnd(rows, width), rnd(rows, sum(parts))


def check(ad, ids, x, y, got):
    want, size, at = y.double(), torch.zeros_like(y, dtype=torch.float64), 0
    rank, width = ad.rank, x.shape[1]
    for a in set(ids.tolist()):
        if not 0 <= a < ad.slots:
            continue
        rows, at = (ids == a).nonzero()[:, 0], 0
        for i, n in enumerate(ad.parts):
            d, u = ad.down[a, i * rank : (i + 1) * rank].double(), ad.up[a, at : at + n].double()
            s = float(ad.scale[a])
            want[rows, at : at + n] += s * (x[rows].double() @ d.t()) @ u.t()
            size[rows, at : at + n] += s * (x[rows].double().abs() @ d.abs().t()) @ u.abs().t()
            at += n
    eps = torch.finfo(y.dtype).eps / 2
    inner = 2.0 ** -16 if y.dtype == torch.bfloat16 else 0.0
    bound = eps * want.abs() + (1 + eps) * ((width + rank + 3) * 2.0 ** -23 + inner) * size + 2.0 ** -23 * want.abs()
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max()
    rest = ~((ids >= 0) & (ids < ad.slots))
    assert torch.equal(got[rest], y[rest])


SHAPES = [
    # rows, width, parts, rank, slots, dtype
    (1, 2048, (2048, 1024, 1024), 16, 1, torch.bfloat16),
    (64, 2048, (2048,), 16, 48, torch.bfloat16),
    (37, 1536, (1792, 896, 768), 24, 5, torch.bfloat16),
    (129, 256, (512, 512), 8, 3, torch.bfloat16),
    (300, 2048, (2048, 1024, 1024), 64, 2, torch.bfloat16),
    (700, 6144, (2048,), 40, 3, torch.bfloat16),
    (200, 512, (96, 40, 8, 200), 128, 2, torch.bfloat16),  # more inner values than the wide form takes
    (17, 72, (33, 7), 8, 2, torch.bfloat16),  # parts that end inside a group, and off eight columns
    (150, 40, (65,), 16, 4, torch.bfloat16),
    (20, 61, (50, 14), 16, 3, torch.bfloat16),  # rows that cannot be read in 16 bytes
    (3, 8, (1,), 8, 2, torch.bfloat16),
    (40, 2048, (1792, 896, 768), 8, 2, torch.float32),
    (161, 1100, (130, 3), 56, 7, torch.float32),
    (1, 1, (5,), 8, 1, torch.float32),
]


@pytest.mark.parametrize("rows,width,parts,rank,slots,dtype", SHAPES)
@pytest.mark.parametrize("tile_rows", [None, 16, 128])
def test_against_the_formula(ops, rows, width, parts, rank, slots, dtype, tile_rows):
    ad, ids, x, y = make(ops, rows, width, parts, rank, slots, dtype)
    plan = ops.plan_adapters(ids, slots, tile_rows)
    out = torch.full_like(y, float("nan"))
    assert ops.add_adapters(y, x, ad, plan, out=out) is out
    check(ad, ids, x, y, out)
    again = ops.add_adapters(y.clone(), x, ad, plan)  # over y itself
    assert torch.equal(again, out)


@pytest.mark.parametrize("rows,width,parts,rank", [
    (1300, 256, (512, 520, 40), 16), (1300, 264, (24, 96, 130), 8), (2500, 72, (70,), 24), (300, 512, (4200,), 32), (999, 2048, (2048, 1024, 1024), 16),
    (1000, 136, (2048,), 32), (257, 64, (128,), 8), (400, 512, (96, 40, 8, 200), 128)])
def test_portions_in_either_form(ops, rows, width, parts, rank):
    """Many rows of few adapters: at each rank enough of them, or columns, for whole tiles of 128, and fewer."""
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-1, 3, (5,), generator=g).repeat_interleave(rows // 5 + 1)[:rows]
    ids[rows // 2] = 2
    ad, ids, x, y = make(ops, rows, width, parts, rank, 3, torch.bfloat16, seed=rows, ids=ids)
    got = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 3), out=torch.empty_like(y))
    check(ad, ids, x, y, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_and_what_lies_beside_them(ops, dtype):
    ad, ids, x, y = make(ops, 50, 128, (64, 32), 16, 3, dtype, seed=4)
    for pad in (8, 3):
        wide_x = torch.full((50, 128 + pad), float("nan"), dtype=dtype, device="cuda")
        wide_y = torch.full((50, 96 + pad), float("nan"), dtype=dtype, device="cuda")
        wide_x[:, :128], wide_y[:, :96] = x, y
        plan = ops.plan_adapters(ids, 3)
        got = ops.add_adapters(wide_y[:, :96], wide_x[:, :128], ad, plan)
        check(ad, ids, x, y, got)
        assert wide_y[:, 96:].isnan().all()


def test_a_row_s_result_does_not_depend_on_the_others(ops):
    ad, ids, x, y = make(ops, 90, 512, (256, 64), 16, 4, torch.bfloat16, seed=2)
    whole = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 4), out=torch.empty_like(y))
    perm = torch.randperm(90, device="cuda")
    mixed = ops.add_adapters(y[perm], x[perm], ad, ops.plan_adapters(ids[perm].contiguous(), 4))
    assert torch.equal(mixed, whole[perm])
    for r in (0, 41, 89):
        one = ops.add_adapters(y[r : r + 1].clone(), x[r : r + 1], ad, ops.plan_adapters(ids[r : r + 1], 4))
        assert torch.equal(one[0], whole[r])


@pytest.mark.parametrize("rows", [1, 31, 128, 1500, 4099])
@pytest.mark.parametrize("slots", [1, 7, 1500])
def test_plan_covers_every_row_once(ops, rows, slots):
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-1, slots, (rows,), generator=g).to("cuda", torch.int32)
    plan = ops.plan_adapters(ids, slots)
    ids, covered = ids.tolist(), []
    for order, (slot, count, _, _) in zip(plan.order.tolist(), plan.tiles.tolist()):
        assert all(ids[r] == slot for r in order[:count]) and all(r == -1 for r in order[count:])
        covered += order[:count]
    assert sorted(covered) == list(range(rows))


def test_ids_out_of_range_are_rows_without_an_adapter(ops):
    from inference_engine_b200 import kernels as K

    ids = torch.tensor([0, 3, -2, 1, -1, 2 ** 31 - 1, 2, 2])
    ad, ids, x, y = make(ops, 8, 64, (64,), 8, 3, torch.bfloat16, ids=ids)
    K.check_status()
    got = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 3), out=torch.empty_like(y))
    check(ad, ids, x, y, got)
    assert K.check_status() == 2  # a token position or id out of range
    ops.plan_adapters(torch.tensor([-1, 0, 2], dtype=torch.int32, device="cuda"), 3)
    assert K.check_status() == 0


def test_nothing_to_do(ops):
    ad, ids, x, y = make(ops, 0, 64, (64,), 8, 3, torch.bfloat16, ids=torch.zeros(0))
    assert ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 3)).shape == (0, 64)
    ad, ids, x, y = make(ops, 5, 64, (64,), 8, 3, torch.bfloat16, ids=torch.full((5,), -1))
    assert torch.equal(ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 3), out=torch.empty_like(y)), y)


def test_load_and_clear(ops):
    for dtype in (torch.bfloat16, torch.float32):
        ad = ops.make_adapters(3, 64, (32, 16), 12, dtype, "cuda")
        assert ad.rank == 16
        g = torch.Generator(device="cuda").manual_seed(1)
        d, u = torch.randn(5, 64, generator=g, device="cuda"), torch.randn(16, 5, generator=g, device="cuda")
        ad.load(1, [None, (d, u)], 0.25)
        x = torch.randn(4, 64, generator=g, device="cuda").to(dtype)
        y = torch.randn(4, 48, generator=g, device="cuda").to(dtype)
        ids = torch.tensor([1, 0, 2, 1], dtype=torch.int32, device="cuda")
        plan = ops.plan_adapters(ids, 3)
        got = ops.add_adapters(y, x, ad, plan, out=torch.empty_like(y))
        check(ad, ids, x, y, got)
        assert torch.equal(got[:, :32], y[:, :32]) and torch.equal(got[1:3], y[1:3]) and not torch.equal(got[0], y[0])
        ad.clear(1)
        assert torch.equal(ops.add_adapters(y, x, ad, plan, out=torch.empty_like(y)), y)


def test_infinities_and_nan_stay_in_their_rows(ops):
    ad, ids, x, y = make(ops, 20, 128, (64,), 16, 2, torch.bfloat16, seed=5, ids=torch.arange(20) % 2)
    clean = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 2), out=torch.empty_like(y))
    x[3, 7], x[6, 100] = float("nan"), float("inf")
    got = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 2), out=torch.empty_like(y))
    rest = torch.ones(20, dtype=torch.bool, device="cuda")
    rest[[3, 6]] = False
    assert torch.equal(got[rest], clean[rest]) and got[3].isnan().all()
    assert not got[6].isfinite().any()


def test_recorded_and_on_another_stream(ops):
    ad, ids, x, y = make(ops, 70, 256, (128, 64), 16, 5, torch.bfloat16, seed=7)
    want = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 5), out=torch.empty_like(y))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 5), out=torch.empty_like(y))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(y)
    with torch.cuda.graph(graph):
        ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 5), out=out)
    for k in range(3):  # other rows and other adapters of the rows through the same graph
        ids.copy_(ids.roll(1))
        x.copy_(x.roll(3, 0))
        graph.replay()
        check(ad, ids, x, y, out)


def test_chained_launches(ops):
    from inference_engine_b200 import kernels as K

    ad, ids, x, y = make(ops, 64, 512, (512,), 16, 20, torch.bfloat16, seed=8)

    def layers():
        plan, h = ops.plan_adapters(ids, 20), x
        for _ in range(6):
            h = ops.add_adapters(y, h, ad, plan, out=torch.empty_like(y))
        return h

    want = layers()
    K.set_early_start(True)
    try:
        got = layers()
        torch.cuda.synchronize()
    finally:
        K.set_early_start(False)
    assert torch.equal(got, want)


def test_calls_on_two_streams_at_once(ops):
    """Portions of both kinds of part beside one another: neither waits for what the other holds."""
    made = [make(ops, 1400, 512, parts, rank, 3, torch.bfloat16, seed=rank, ids=torch.arange(1400) // 500)
            for parts, rank in (((512, 256, 256), 64), ((2048,), 40), ((256, 256), 128), ((512,), 32))]
    plans = [ops.plan_adapters(m[1], 3) for m in made]
    want = [ops.add_adapters(y, x, ad, plan, out=torch.empty_like(y)) for (ad, _, x, y), plan in zip(made, plans)]
    streams = [torch.cuda.Stream() for _ in made]
    outs = [[torch.empty_like(w) for _ in range(6)] for w in want]
    torch.cuda.synchronize()
    for i in range(6):
        for s, (ad, _, x, y), plan, out in zip(streams, made, plans, outs):
            with torch.cuda.stream(s):
                ops.add_adapters(y, x, ad, plan, out=out[i])
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        assert all(torch.equal(o, w) for o in out)


def test_two_recorded_steps(ops):
    """Each has a plan and a workspace of its own, and sees the ids and rows of its replay."""
    ad, ids, x, y = make(ops, 1300, 256, (512, 64), 64, 4, torch.bfloat16, seed=9, ids=torch.arange(1300) // 400)
    ops.add_adapters(y, x, ad, ops.plan_adapters(ids, 4), out=torch.empty_like(y))
    steps = []
    for n in (1300, 700):
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(y[:n])
        with torch.cuda.graph(graph):
            plan = ops.plan_adapters(ids[:n], 4)
            ops.add_adapters(y[:n], x[:n], ad, plan, out=out)
        steps.append((graph, out, plan, n))
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(2):
        ids.copy_(torch.randint(-1, 4, (1300,), generator=g, device="cuda").sort().values)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        for graph, out, _, n in steps:
            graph.replay()
        for graph, out, _, n in steps:
            check(ad, ids[:n], x[:n], y[:n], out)


@pytest.mark.parametrize("rows,rank,slots", [(60, 16, 20), (90, 24, 4), (700, 64, 5), (40, 8, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("early", [None, True])
def test_steps_behind_one_another_read_their_own_plan_and_rows(ops, rows, rank, slots, dtype, early):
    """Nothing waits between the steps, whose plans lie at one address and whose rows are written over those of the step before."""
    from inference_engine_b200 import kernels as K

    ad, _, _, _ = make(ops, rows, 264, (264, 9), rank, slots, dtype, seed=rows)
    g = torch.Generator(device="cuda").manual_seed(2)
    steps = [(torch.randint(-1, slots, (rows,), generator=g, device="cuda", dtype=torch.int32), torch.randn(rows, 264, generator=g, device="cuda").to(dtype),
              torch.randn(rows, 273, generator=g, device="cuda").to(dtype)) for _ in range(12)]
    want = []
    for ids, x, y in steps:
        once = ops.add_adapters(y, x, ad, ops.plan_adapters(ids, slots), out=torch.empty_like(y))
        check(ad, ids, x, y, once)
        h = once[:, :264].contiguous()
        torch.cuda.synchronize()
        want.append(ops.add_adapters(y, h, ad, ops.plan_adapters(ids, slots), out=torch.empty_like(y)))
        torch.cuda.synchronize()
    if early:
        K.set_early_start(True)
    try:
        got, wide = [], torch.empty(rows, 280, dtype=dtype, device="cuda")[:, :273]
        for ids, x, y in steps:
            plan = ops.plan_adapters(ids, slots)
            ops.add_adapters(y, x, ad, plan, out=wide)
            got.append(ops.add_adapters(y, wide[:, :264], ad, plan, out=torch.empty_like(y)))
            del plan
    finally:
        if early:
            K.set_early_start(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_without_early_starts(ops):
    from inference_engine_b200 import kernels as K

    made = [(slots, make(ops, rows, 512, (512,), rank, slots, torch.bfloat16, seed=8)) for rows, rank, slots in ((64, 16, 20), (900, 64, 3))]

    def results():
        return [ops.add_adapters(y, x, ad, ops.plan_adapters(ids, slots), out=torch.empty_like(y)) for slots, (ad, ids, x, y) in made]

    K.set_early_start(True)
    want = results()
    K.set_early_start(False)
    got, graph = results(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = results()
    graph.replay()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, recorded))


@pytest.mark.parametrize("rows,width,parts,rank,slots,used", [
    (1300, 256, (512, 520, 40), 64, 700, 3), (300, 72, (4200, 130), 40, 300, 300), (520, 128, (256,), 64, 4096, 1), (2000, 64, (96, 4000), 128, 48, 5),
    (700, 128, (40000,), 64, 2, 2)])
def test_portions_beside_slots_that_nobody_uses(ops, rows, width, parts, rank, slots, used):
    """Tiles that could have rows and do not, up to many times those that do; and runs of many columns."""
    g = torch.Generator().manual_seed(rows)
    of = torch.randperm(slots, generator=g)[:used]
    ids = of[torch.arange(rows) * used // rows]
    ids[rows // 3] = -1
    ad, ids, x, y = make(ops, rows, width, parts, rank, slots, torch.bfloat16, seed=rows, ids=ids)
    plan = ops.plan_adapters(ids, slots)
    assert plan.tile_rows == 128
    live = plan.tiles[:, 1].gt(0)
    assert plan.tiles[0, 2] == live.sum() and live[: live.sum()].all()
    got = ops.add_adapters(y, x, ad, plan, out=torch.empty_like(y))
    check(ad, ids, x, y, got)


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 56, 64, 72, 128])
@pytest.mark.parametrize("rows,used,slots", [(1, 1, 40), (16, 16, 16), (64, 48, 48), (40, 3, 9)])
def test_clusters_of_every_size_at_every_rank(ops, rank, rows, used, slots):
    g = torch.Generator().manual_seed(rank)
    ids = torch.randperm(slots, generator=g)[:used][torch.arange(rows) % used]
    for width, parts in ((264, (512, 33)), (1024, (2600,)), (72, (1032, 1032, 8, 64))):
        ad, at, x, y = make(ops, rows, width, parts, rank, slots, torch.bfloat16, seed=rank, ids=ids)
        check(ad, at, x, y, ops.add_adapters(y, x, ad, ops.plan_adapters(at, slots, 16), out=torch.empty_like(y)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,rank,slots,tile_rows", [(70, 16, 3, 16), (300, 64, 2, 128), (300, 8, 2, 128), (5, 128, 1, 16)])
def test_rows_without_an_adapter_are_copied_or_left(ops, dtype, rows, rank, slots, tile_rows):
    g = torch.Generator().manual_seed(rows)
    ids = torch.where(torch.rand(rows, generator=g) < 0.7, torch.full((rows,), -1), torch.randint(0, slots, (rows,), generator=g))
    for width, parts in ((128, (700, 70)), (72, (33,)), (2048, (1024,))):
        ad, at, x, y = make(ops, rows, width, parts, rank, slots, dtype, seed=rank, ids=ids)
        y[ids == -1] = float("nan")
        plan = ops.plan_adapters(at, slots, tile_rows)
        wide = torch.full((rows, y.shape[1] + 5), 7.0, dtype=dtype, device="cuda")
        got = ops.add_adapters(y, x, ad, plan, out=wide[:, : y.shape[1]])
        none = (ids == -1).cuda()
        assert got[none].isnan().all() and got[~none].isfinite().all() and (wide[:, y.shape[1] :] == 7).all()
        check(ad, at[~none], x[~none], y[~none], got[~none])
        assert torch.equal(ops.add_adapters(y.clone(), x, ad, plan)[~none], got[~none])
