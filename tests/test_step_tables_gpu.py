"""ops.step_tables against the same rules written as loops, and against the host's cache manager."""
import numpy as np
import pytest
import torch

from imparo_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(lengths, counts, free, held, page, width, n_tokens, parent=None, shared=None):
    items = len(lengths)
    table = np.full((items, width), -1, dtype=np.int32)
    positions, item_of, slots = np.full(n_tokens, -1), np.zeros(n_tokens, dtype=np.int64), np.full(n_tokens, -1)
    row_start, taken, t = [], 0, 0
    for r in range(items):
        row_start.append(t)
        for b in range(width):
            src = held[parent[r]] if parent is not None and parent[r] >= 0 and b < shared[r] // page else held[r]
            if b < len(src):
                table[r, b] = src[b]
        for pos in range(lengths[r], lengths[r] + counts[r]):
            b = pos // page
            if table[r, b] < 0:
                table[r, b] = free[taken]
                taken += 1
            positions[t], item_of[t], slots[t] = pos, r, int(table[r, b]) * page + pos % page
            t += 1
    row_start.append(t)
    return table, positions, item_of, row_start, slots, [taken]


def device_call(lengths, counts, free, held, page, n_pages, width, n_tokens, parent=None, shared=None, status=None):
    i32 = lambda v: torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)
    new = lambda *shape, dtype=torch.int32: torch.full(shape, 12345, dtype=dtype, device=DEV)
    items = len(lengths)
    outs = [new(items, width), new(n_tokens), new(n_tokens), new(items + 1), new(n_tokens, dtype=torch.int64), new(1)]
    status = ops.new_status(DEV) if status is None else status
    ops.step_tables(i32(lengths), i32(counts), i32(free), i32(held), page, n_pages, *outs, status,
                    parent=None if parent is None else i32(parent), shared=None if shared is None else i32(shared))
    return outs, status


def check(*args, **kw):
    lengths, counts, free, held, page, n_pages, width, n_tokens = args
    outs, status = device_call(*args, **kw)
    ops.read_status(status)
    for got, want, name in zip(outs, plain(lengths, counts, free, held, page, width, n_tokens, **kw),
                               ("table", "positions", "item_of_token", "row_start", "slots", "taken")):
        assert np.array_equal(got.cpu().numpy(), np.asarray(want)), name


def draw(seed, items, most_held, most_new, page, forked=False, holes=False, spare_tokens=0, zero_counts=True):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, most_held + 1, items)
    counts = rng.integers(0 if zero_counts else 1, most_new + 1, items)
    parent, shared = np.full(items, -1), np.zeros(items, dtype=np.int64)
    if forked:
        for r in range(items):
            if r % 3:
                parent[r] = r - r % 3
                shared[r] = rng.integers(0, lengths[parent[r]] + 1)
                lengths[r] = shared[r] // page * page if rng.random() < 0.5 else shared[r]
    width = int((-(-(lengths + counts) // page)).max()) + 2
    need = int((-(-(lengths + counts) // page)).sum()) + 1
    pages = rng.permutation(2 * need + 3)
    held = np.full((items, max(1, int((-(-lengths // page)).max()) + 1)), -1)
    at = 0
    for r in range(items):
        n = -(-int(lengths[r]) // page)
        if parent[r] >= 0:
            continue
        held[r, :n] = pages[at:at + n]
        at += n
        if holes and n > 2:
            held[r, :n - 2] = -1                                   # a window has passed these
    return (lengths, counts, np.sort(pages[at:]), held, page, 2 * need + 3, width, int(counts.sum()) + spare_tokens), \
        (dict(parent=parent, shared=shared) if forked else {})


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("items,most_held,most_new", [(1, 0, 1), (1, 100, 300), (7, 50, 1), (40, 3000, 70), (300, 500, 5), (1500, 40, 3), (5000, 9, 2)])
def test_random_steps(items, most_held, most_new, page):
    args, kw = draw(items + page, items, most_held, most_new, page)
    check(*args, **kw)


@pytest.mark.parametrize("page", [1, 16, 32])
@pytest.mark.parametrize("items", [3, 50, 1300])
def test_forked_items(items, page):
    args, kw = draw(items, items, 700, 40, page, forked=True)
    check(*args, **kw)


def test_holes_and_spare_tokens():
    args, kw = draw(3, 60, 900, 33, 16, holes=True, spare_tokens=77)
    check(*args, **kw)


def test_no_new_tokens():
    check(np.array([5, 0, 32]), np.array([0, 0, 0]), np.array([9]), np.array([[1, -1], [-1, -1], [2, 3]]), 16, 10, 3, 4)


def test_blocks_mapped_ahead_are_kept():
    """A page reserved for new positions beforehand is not taken again."""
    check(np.array([16, 10]), np.array([40, 8]), np.array([7, 8, 9]), np.array([[0, 1, -1, 2], [3, -1, -1, -1]]), 16, 10, 4, 48)


def test_as_the_cache_manager_hands_pages_out():
    from imparo_b200.cache import CacheManager
    from imparo_b200.parts.spec import PagedKV
    rng = np.random.default_rng(2)
    cm = CacheManager([(0, (PagedKV(1, 16, None),))], 16, 400, 20)
    for r in range(12):
        cm.add(r)
    width = 40
    for _ in range(12):
        live = [r for r in range(12) if rng.random() < 0.7]
        counts = [int(rng.integers(1, 40)) for _ in live]
        lengths = [cm.cached(r) for r in live]
        held = np.stack([cm.table(r, 0, width) for r in live])
        used = {p for r in range(12) for p in cm.table(r, 0, width) if p >= 0}
        free = [p for p in range(400) if p not in used]
        outs, status = device_call(lengths, counts, free, held, 16, 400, width, sum(counts))
        ops.read_status(status)
        for r, c in zip(live, counts):
            cm.reserve(r, c)
        assert np.array_equal(outs[0].cpu().numpy(), np.stack([cm.table(r, 0, width) for r in live]))
        for r, c in zip(live, counts):
            cm.commit(r, c)


def test_slots_beyond_32_bits():
    check(np.array([100]), np.array([3]), np.array([2000000001]), np.array([[2000000000]]), 101, 2000000005, 2, 3)


@pytest.mark.parametrize("what", ["free list too short", "table too narrow", "tokens too few", "negative length", "negative count",
                                  "page out of range", "free page out of range", "parent out of range"])
def test_what_does_not_fit_is_reported(what):
    lengths, counts, free, held = np.array([20, 5, 0]), np.array([30, 3, 2]), np.array([5, 6, 7, 8, 9]), np.array([[0, 1], [2, -1], [-1, -1]])
    n_pages, width, n_tokens, kw = 10, 4, 35, {}
    if what == "free list too short":
        free = free[:2]
    elif what == "table too narrow":
        width = 3
    elif what == "tokens too few":
        n_tokens = 33
    elif what == "negative length":
        lengths = np.array([20, -5, 0])
    elif what == "negative count":
        counts = np.array([30, -3, 2])
    elif what == "page out of range":
        held = np.array([[0, 10], [2, -1], [-1, -1]])
    elif what == "free page out of range":
        free = np.array([5, 600, 7, 8, 9])
    else:
        kw = dict(parent=[-1, 3, -1], shared=[0, 16, 0])
    outs, status = device_call(lengths, counts, free, held, 16, n_pages, width, n_tokens, **kw)
    with pytest.raises(ops.KernelError):
        ops.read_status(status)
    table, slots = outs[0].cpu().numpy(), outs[4].cpu().numpy()
    assert slots.max() < n_pages * 16 and slots.min() >= -1 and table.min() >= -1
    if what == "tokens too few":                                   # the others are as ever
        assert np.array_equal(table, plain(lengths, counts, free, held, 16, width, 35)[0])


def test_captured_and_replayed():
    args, _ = draw(1, 20, 300, 4, 16, zero_counts=False)
    lengths, counts, free, held, page, n_pages, width, n_tokens = args
    i32 = lambda v: torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)
    ins = [i32(x) for x in (lengths, counts, free, held)]
    outs = [i32(np.zeros((20, width))), i32(np.zeros(n_tokens)), i32(np.zeros(n_tokens)), i32(np.zeros(21)),
            torch.zeros(n_tokens, dtype=torch.int64, device=DEV), i32([0])]
    status = ops.new_status(DEV)
    run = lambda: ops.step_tables(*ins, page, n_pages, *outs, status)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    ins[0].copy_(i32(np.maximum(lengths - 1, 0)))
    graph.replay()
    for got, want in zip(outs, plain(np.maximum(lengths - 1, 0), counts, free, held, page, width, n_tokens)):
        assert np.array_equal(got.cpu().numpy(), np.asarray(want))


@pytest.mark.parametrize("change,code,where", [
    (dict(free=[5, 6]), 5, 63), (dict(width=3), 5, 61), (dict(n_tokens=33), 5, 65), (dict(lengths=[20, -5, 0]), 5, 60),
    (dict(counts=[30, -3, 2]), 5, 60), (dict(parent=[-1, 3, -1], shared=[0, 16, 0]), 5, 62), (dict(parent=[-1, 0, -1], shared=[0, 16, 0]), 5, 66),
    (dict(held=[[0, 10], [2, -1], [-1, -1]]), 2, 64), (dict(free=[5, 600, 7, 8, 9]), 2, 63)])
def test_what_does_not_fit_is_named(change, code, where):
    args = dict(lengths=[20, 5, 0], counts=[30, 3, 2], free=[5, 6, 7, 8, 9], held=[[0, 1], [2, -1], [-1, -1]], page=16, n_pages=10, width=4, n_tokens=35)
    _, status = device_call(**{**args, **change})
    assert status.tolist()[:2] == [code, where]
    with pytest.raises(ops.KernelError, match="step's description" if code == 5 else "cache page out of range"):
        ops.read_status(status)


@pytest.mark.parametrize("between", [False, True])
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kernels_right_behind_read_the_new_tables(dtype, graph, between):
    """The cache writer and the attention, launched behind the tables with nothing in between (or one more kernel of the chain): the
    arrays hold another step's description before, as valid as the new one."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    nh, nkv, hd, page, items, width, n_pages = 8, 2, 64, 16, 64, 40, 64 * 40
    i32 = lambda v: torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)
    steps = []
    for seed in (0, 1):
        rng = np.random.default_rng(seed)
        lengths, counts = rng.integers(0, 600, items), np.ones(items, dtype=np.int64)
        pages = rng.permutation(n_pages)
        held = np.full((items, width), -1)
        at = 0
        for r in range(items):
            n = -(-int(lengths[r]) // page)
            held[r, :n] = pages[at:at + n]
            at += n
        free = pages[at:at + items]
        made = plain(lengths, counts, free, held, page, width, items)
        steps.append(([i32(x) for x in (lengths, counts, free, held)], i32(made[0]), i32(made[1])))
    item_of, row_start, slots, taken = i32(np.zeros(items)), i32(np.zeros(items + 1)), torch.zeros(items, dtype=torch.int64, device=DEV), i32([0])
    table, positions = i32(np.zeros((items, width))), i32(np.zeros(items))
    status = ops.new_status(DEV)
    draw = lambda *shape: torch.randn(*shape, device=DEV, generator=gen).to(dtype)
    qkv, first_k, first_v = draw(items, (nh + 2 * nkv) * hd), draw(n_pages, page, nkv * hd), draw(n_pages, page, nkv * hd)
    inv_freq = 10000.0 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float32) / (hd // 2))
    q, out, k, v = torch.empty(items, nh * hd, dtype=dtype, device=DEV), torch.empty(items, nh * hd, dtype=dtype, device=DEV), first_k.clone(), first_v.clone()
    chunk, n_splits = ops.split_plan(items, nkv, width * page)
    acc, ml = torch.empty(items * nh * n_splits * hd, device=DEV), torch.empty(items * nh * n_splits * 2, device=DEV)
    some, weight, normed = torch.randn(4, 64, device=DEV, generator=gen), torch.ones(64, device=DEV), torch.empty(4, 64, device=DEV)

    def reads(table, positions, item_of):
        ops.qk_norm_rope_store(qkv, positions, item_of, None, None, inv_freq, hd, 1e-6, q, k, v, table, page, n_pages, nh, nkv, hd, status)
        assert ops.paged_attention_split(q, k, v, positions, item_of, table, page, n_pages, None, hd ** -0.5, out, acc, ml, chunk, n_splits, nh,
                                         nkv, hd, status)

    def step(which):
        ops.step_tables(*steps[which][0], page, n_pages, table, positions, item_of, row_start, slots, taken, status)
        if between:
            ops.rmsnorm(some, weight, 1e-6, normed)
        reads(table, positions, item_of)

    def whole(run):
        k.copy_(first_k)
        v.copy_(first_v)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        ops.read_status(status)
        return q.clone(), out.clone(), k.clone(), v.clone()

    order = i32(np.arange(items))
    want = [whole(lambda: reads(steps[w][1], steps[w][2], order)) for w in (0, 1)]
    assert not torch.equal(want[0][1], want[1][1])
    graphs = []
    for w in (0, 1):
        step(w)
        torch.cuda.synchronize()
        if graph:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                step(w)
    for n in range(12):
        w = n % 2
        for got, expected in zip(whole(graphs[w].replay if graph else lambda: step(w)), want[w]):
            assert torch.equal(got, expected)


def test_refusals():
    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    names = ("lengths", "counts", "free_pages", "held", "page_size", "n_pages", "table", "positions", "item_of_token", "row_start", "slots",
             "taken", "status")
    good = dict(zip(names, (i32(3), i32(3), i32(9), i32(3, 4), 16, 100, i32(3, 5), i32(7), i32(7), i32(4),
                            torch.zeros(7, dtype=torch.int64, device=DEV), i32(1), ops.new_status(DEV))))
    whole = i32(40)
    for change in (dict(lengths=i32(2)), dict(counts=i32(3).long()), dict(held=i32(2, 4)), dict(held=i32(12)), dict(table=i32(3, 5).float()),
                   dict(slots=i32(7)), dict(slots=torch.zeros(6, dtype=torch.int64, device=DEV)), dict(item_of_token=i32(6)),
                   dict(row_start=i32(3)), dict(parent=i32(3)), dict(shared=i32(3)), dict(page_size=0), dict(n_pages=0),
                   dict(table=whole[:15].view(3, 5), held=whole[10:22].view(3, 4)), dict(lengths=i32(3).cpu()),
                   dict(table=i32(3, 8)[:, :5])):
        with pytest.raises(ops.KernelError):
            ops.step_tables(**{**good, **change})


def test_pages_that_do_not_exist_are_left_out_of_the_table():
    """Held ones of past positions too, and negative ones of the free list; the rest of the step is as ever."""
    outs, status = device_call(np.array([40, 5]), np.array([10, 3]), np.array([-5, 6, 7]), np.array([[3, 99, -1, -1], [2, -1, -1, 77]]), 16, 10, 4, 13)
    with pytest.raises(ops.KernelError):
        ops.read_status(status)
    assert outs[0].tolist() == [[3, -1, -1, 6], [2, -1, -1, -1]] and outs[5].tolist() == [2]
    assert outs[4].tolist() == [-1] * 8 + [96, 97] + [37, 38, 39]
    assert outs[1].tolist() == list(range(40, 50)) + [5, 6, 7]


def test_new_positions_never_go_to_a_parents_page():
    """More shared positions than the item holds: reported, and its new ones take a page of their own."""
    outs, status = device_call(np.array([40, 20]), np.array([1, 2]), np.array([8, 9]), np.array([[3, 4, 5], [-1, -1, -1]]), 16, 10, 3, 3,
                               parent=[-1, 0], shared=[0, 40])
    with pytest.raises(ops.KernelError):
        ops.read_status(status)
    assert outs[0].tolist() == [[3, 4, 5], [3, 8, -1]] and outs[4].tolist() == [5 * 16 + 8, 8 * 16 + 4, 8 * 16 + 5]
