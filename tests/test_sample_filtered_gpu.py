"""ops.sample_filtered against the definition in 80-bit sums: the same token and the same number of tokens left, everywhere."""
import numpy as np
import pytest
import torch

from imparo_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain_pick(logits, temperature, u, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, tokens left).  logits: the kernel's inputs as 64-bit numbers."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    live = np.flatnonzero(x > -np.inf)
    if live.size == 0:
        return 0, 0
    top = x.max()
    if not temperature > 0:
        return int(live[x[live].argmax()]), 1
    order = live[np.lexsort((live, -x[live]))]
    if top_k > 0:
        order = order[:top_k]

    def weights(at):
        with np.errstate(invalid="ignore", under="ignore"):
            return np.where(x[at] == top, 1.0, np.exp((x[at] - top) / np.float64(temperature))).astype(np.longdouble)
    w = weights(order)
    if top_p < 1:
        before = np.concatenate([[np.longdouble(0)], np.cumsum(w)[:-1]])
        stay = max(1, int((before < np.longdouble(top_p) * w.sum()).sum()))
        order, w = order[:stay], w[:stay]
    if min_p > 0:
        order = order[:max(1, int((w >= np.longdouble(min_p)).sum()))]
    rising = np.sort(order)
    sums = np.cumsum(weights(rising))
    return int(rising[min(np.searchsorted(sums, np.longdouble(u) * sums[-1], side="right"), len(rising) - 1)]), len(rising)


def check(logits, temperature, uniform, top_k=None, top_p=None, min_p=None, call=ops.sample_filtered):
    n = logits.shape[0]
    f32 = lambda v: None if v is None else torch.tensor(np.asarray(v, dtype=np.float32), device=DEV)
    i32 = lambda v: None if v is None else torch.tensor(np.asarray(v, dtype=np.int32), device=DEV)
    out, kept = (torch.full((n + 2,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    call(logits, f32(temperature), f32(uniform), out, top_k=i32(top_k), top_p=f32(top_p), min_p=f32(min_p), kept=kept)
    x = logits.double().cpu().numpy()
    value = lambda v, r, default: default if v is None else np.asarray(v, dtype=np.float32)[r] if not np.asarray(v).dtype.kind == "i" else int(v[r])
    want = [plain_pick(x[r], np.float32(temperature[r]), np.float32(uniform[r]), value(top_k, r, 0), value(top_p, r, 1.0), value(min_p, r, 0.0))
            for r in range(n)]
    got = list(zip(out.tolist()[:n], kept.tolist()[:n]))
    assert got == want
    assert out.tolist()[n:] == [-7, -7] and kept.tolist()[n:] == [-7, -7]
    return got


def settings(rng, n, vocab):
    """Every filter alone, none, all together, and greedy rows."""
    which = rng.integers(0, 7, n)
    t = rng.uniform(0.3, 2.0, n).astype(np.float32)
    t[which == 6] = 0
    k = np.where(np.isin(which, (1, 4)), np.exp(rng.uniform(0, np.log(vocab + 1), n)), 0).astype(np.int32)
    p = np.where(np.isin(which, (2, 4)), rng.uniform(0.05, 0.999, n), 1.0).astype(np.float32)
    m = np.where(np.isin(which, (3, 4)), np.exp(rng.uniform(np.log(1e-6), 0, n)), 0).astype(np.float32)
    u = (rng.integers(0, 1 << 24, n) / float(1 << 24)).astype(np.float32)
    return t, u, k, p, m


@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 2048, 2049, 4097, 32003, 65536, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_rows(vocab, dtype):
    rng = np.random.default_rng(vocab)
    n = 24
    logits = torch.tensor(rng.standard_normal((n, vocab)) * rng.uniform(0.5, 5, (n, 1)), dtype=dtype, device=DEV)
    t, u, k, p, m = settings(rng, n, vocab)
    check(logits, t, u, k, p, m)


@pytest.mark.parametrize("n", [1, 2, 7, 148, 300])
def test_many_rows(n):
    rng = np.random.default_rng(n)
    logits = torch.tensor(rng.standard_normal((n, 5003)) * 3, dtype=torch.float32, device=DEV)
    check(logits, *settings(rng, n, 5003))


def test_vocabulary_beyond_shared_memory():
    rng = np.random.default_rng(5)
    logits = torch.tensor(rng.standard_normal((7, 400001)) * 2, dtype=torch.float32, device=DEV)
    check(logits, [1.0] * 7, [0.3, 0.9, 0.5, 0.1, 0.7, 0.2, 0.99], [0, 5, 0, 1000, 300000, 0, 0], [1, 1, 0.9, 0.8, 0.5, 1, 0.01],
          [0, 0, 0, 0, 0, 1e-3, 0])


@pytest.mark.parametrize("vocab", [140000, 140001, 140002, 140003])
def test_picks_among_the_last_entries_of_a_long_row(vocab):
    """The row's end is no multiple of four, and parts of its last stretch are empty: each entry is weighed once."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    x[:, -9:] += 12.0
    u = [1 - 2.0 ** -24, 0.999, 0.97, 0.9, 0.6, 0.3]
    for k, p, m in (([0] * 6, [1.0] * 6, [0.0] * 6), ([0] * 6, [0.99] * 6, [0.0] * 6), ([100000] * 6, [1.0] * 6, [1e-9] * 6)):
        got = check(torch.tensor(x, device=DEV), [1.0] * 6, u, k, p, m)
        assert got[0][0] == vocab - 1 or p[0] < 1


@pytest.mark.parametrize("vocab", [4096, 40000])
def test_equal_logits_stay_by_index(vocab):
    logits = torch.zeros(9, vocab, device=DEV)
    logits[5:, ::2] = -0.0                                         # equal to the others all the same
    half = vocab // 2
    got = check(logits, [1.0] * 9, [0.0, 0.25, 0.5, 0.999, 0.5, 0.25, 0.5, 0.75, 0.0], [0, half, 0, half, 3, 0, half + 1, 0, 1],
                [1, 1, 0.5, 0.25, 1, 0.5, 0.5, 0.125, 1], [0, 0, 0, 0, 0, 1, 0, 0, 0])
    assert got[2] == (vocab // 4, half) and got[8] == (0, 1)


def test_few_levels_many_ties():
    """Logits of eight values, in 16 bits: every border lies among thousands of equal entries."""
    rng = np.random.default_rng(11)
    n, vocab = 64, 50000
    logits = torch.tensor(rng.integers(0, 8, (n, vocab)) * 0.5, dtype=torch.bfloat16, device=DEV)
    check(logits, *settings(rng, n, vocab))


@pytest.mark.parametrize("spread", [1e-6, 1e-3, 30.0, 1e4])
def test_narrow_and_wide_rows(spread):
    """All logits within one bin of the histogram, and nearly all beyond the last one."""
    rng = np.random.default_rng(3)
    n, vocab = 32, 20000
    logits = torch.tensor(7.0 + rng.standard_normal((n, vocab)) * spread, dtype=torch.float32, device=DEV)
    check(logits, *settings(rng, n, vocab))


@pytest.mark.parametrize("temperature", [1e-30, 1e-4, 50.0, 1e30, float("inf")])
def test_extreme_temperatures(temperature):
    rng = np.random.default_rng(4)
    n, vocab = 28, 9000
    logits = torch.tensor(rng.standard_normal((n, vocab)) * 2, dtype=torch.float32, device=DEV)
    t, u, k, p, m = settings(rng, n, vocab)
    check(logits, np.where(t > 0, np.float32(temperature), 0).astype(np.float32), u, k, p, m)


def test_nan_infinities_and_masks():
    rng = np.random.default_rng(6)
    n, vocab = 40, 6001
    x = rng.standard_normal((n, vocab)).astype(np.float32) * 2
    x[:, ::3] = -np.inf
    x[::2, 1::5] = np.nan
    x[3] = -np.inf                                                 # nothing at all
    x[4] = np.nan
    x[5] = -np.inf
    x[5, 4000] = -3e38                                             # one entry left
    x[6, [10, 77, 5000]] = np.inf                                  # these share all the weight
    x[7] = torch.finfo(torch.float32).min                          # masked with the type's lowest value throughout
    x[8] = torch.finfo(torch.float32).min
    x[8, 123] = 1.0
    x[9, 100] = torch.finfo(torch.float32).max
    t, u, k, p, m = settings(rng, n, vocab)
    got = check(torch.tensor(x, device=DEV), t, u, k, p, m)
    assert got[3] == (0, 0) and got[4] == (0, 0) and got[5] == (4000, 1)


@pytest.mark.parametrize("vocab", [900, 70001])
def test_infinite_logits_take_all_the_weight_at_any_temperature(vocab):
    rng = np.random.default_rng(7)
    t, u, k, p, m = settings(rng, 28, vocab)
    x = rng.standard_normal((28, vocab)).astype(np.float32)
    x[:, [5, 300, vocab - 1]] = np.inf
    x = torch.tensor(x, device=DEV)
    want = check(x, t, u, k, p, m)
    i32, f32 = (lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)), (lambda v: torch.tensor(np.asarray(v), dtype=torch.float32, device=DEV))
    for hot in (1e30, np.inf):
        out, kept = i32(np.zeros(28)), i32(np.zeros(28))
        ops.sample_filtered(x, f32(np.where(t > 0, hot, 0)), f32(u), out, top_k=i32(k), top_p=f32(p), min_p=f32(m), kept=kept)
        # (top-k may leave other entries of weight 0, where there are more than three: the same ones at any temperature)
        assert list(zip(out.tolist(), kept.tolist())) == want


def test_single_settings_at_their_limits():
    rng = np.random.default_rng(8)
    vocab = 3001
    row = rng.standard_normal(vocab).astype(np.float32)
    u = np.float32(1) - np.float32(2 ** -24)
    cases = [  # top_k, top_p, min_p, uniform
        (1, 1.0, 0.0, 0.7), (vocab, 1.0, 0.0, 0.7), (vocab + 9, 1.0, 0.0, 0.2), (-3, 1.0, 0.0, 0.7), (0, 0.0, 0.0, 0.7), (0, -1.0, 0.0, 0.3),
        (0, 1e-12, 0.0, 0.7), (0, 1e-40, 0.0, 0.7), (0, float(u), 0.0, 0.7), (0, 2.0, 0.0, 0.7), (0, 1.0, 1.0, 0.7), (0, 1.0, 1.5, 0.7),
        (0, 1.0, -1.0, 0.7), (0, 1.0, 1e-38, 0.7), (50, 0.5, 0.1, 0.0), (50, 0.5, 0.1, float(u)), (0, 1.0, 0.0, 0.0), (0, 1.0, 0.0, float(u)),
        (0, 1.0, 0.0, 1e-30), (2, 0.99, 0.01, 0.5)]
    k, p, m, uu = (np.array(c) for c in zip(*cases))
    check(torch.tensor(np.tile(row, (len(cases), 1)), device=DEV), np.ones(len(cases), dtype=np.float32), uu.astype(np.float32),
          k.astype(np.int32), p.astype(np.float32), m.astype(np.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_apart_and_unaligned(dtype):
    rng = np.random.default_rng(9)
    wide = torch.tensor(rng.standard_normal((12, 5000)) * 2, dtype=dtype, device=DEV)
    for first, vocab in ((0, 4999), (1, 4096), (3, 2500), (7, 33)):
        check(wide[:, first:first + vocab], *settings(rng, 12, vocab))
    check(wide[::3, 5:4005], *settings(rng, 4, 4000))


def test_same_result_every_time_and_beside_other_rows():
    rng = np.random.default_rng(10)
    logits = torch.tensor(rng.standard_normal((40, 65536)) * 2, dtype=torch.float32, device=DEV)
    t, u, k, p, m = settings(rng, 40, 65536)
    first = check(logits, t, u, k, p, m)
    assert check(logits, t, u, k, p, m) == first
    assert check(logits[13:14], t[13:14], u[13:14], k[13:14], p[13:14], m[13:14]) == first[13:14]


def test_captured_and_replayed_on_another_stream():
    rng = np.random.default_rng(12)
    n, vocab = 6, 10007
    logits = torch.tensor(rng.standard_normal((n, vocab)) * 2, dtype=torch.float32, device=DEV)
    t, u, k, p, m = settings(rng, n, vocab)
    args = [torch.tensor(x, device=DEV) for x in (t, u, k, p, m)]
    out, kept = (torch.zeros(n, dtype=torch.int32, device=DEV) for _ in range(2))
    run = lambda: ops.sample_filtered(logits, args[0], args[1], out, top_k=args[2], top_p=args[3], min_p=args[4], kept=kept)
    run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        run()
    for seed in range(3):
        rng = np.random.default_rng(100 + seed)
        logits.copy_(torch.tensor(rng.standard_normal((n, vocab)) * 2, dtype=torch.float32))
        fresh = settings(rng, n, vocab)
        for a, b in zip(args, fresh):
            a.copy_(torch.tensor(b))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        want = [plain_pick(logits[r].double().cpu().numpy(), fresh[0][r], fresh[1][r], int(fresh[2][r]), fresh[3][r], fresh[4][r]) for r in range(n)]
        assert list(zip(out.tolist(), kept.tolist())) == want


@pytest.mark.parametrize("rows", [1, 3, 8, 60])
def test_a_row_of_several_ctas_while_other_kernels_come_and_go(rows):
    """A row's CTAs give one another what they found in their stretches as soon as all of them run, however busy the SMs are."""
    rng = np.random.default_rng(rows)
    vocab = 65536
    logits = torch.tensor(rng.standard_normal((rows, vocab)) * 2, dtype=torch.float32, device=DEV)
    settled = settings(rng, rows, vocab)
    want = check(logits, *settled)
    args = [torch.tensor(x, device=DEV) for x in settled]
    calls = 40
    outs, kepts = ([torch.full((rows,), -7, dtype=torch.int32, device=DEV) for _ in range(calls)] for _ in range(2))
    side, a, small = torch.cuda.Stream(), torch.randn(1024, 1024, device=DEV), torch.randn(1 << 16, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(60):
            a = torch.tanh(a @ a)
            small = small * 0.5 + 1.0
    for out, kept in zip(outs, kepts):
        ops.sample_filtered(logits, args[0], args[1], out, top_k=args[2], top_p=args[3], min_p=args[4], kept=kept)
    torch.cuda.synchronize()
    for out, kept in zip(outs, kepts):
        assert list(zip(out.tolist(), kept.tolist())) == want


def test_no_rows():
    e = torch.empty(0, device=DEV)
    ops.sample_filtered(torch.empty(0, 100, device=DEV), e, e, torch.empty(0, dtype=torch.int32, device=DEV))


def test_refusals():
    logits = torch.zeros(4, 100, device=DEV)
    f, i = torch.ones(4, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    good = dict(logits=logits, temperature=f, uniform=f, out=i)
    for change in (dict(logits=logits.half()), dict(logits=logits[0]), dict(logits=logits.t()), dict(temperature=f.double()),
                   dict(uniform=f[:3]), dict(out=i.long()), dict(top_k=f), dict(top_p=i), dict(min_p=f[:2]), dict(kept=f),
                   dict(temperature=None), dict(uniform=None), dict(logits=logits.cpu()), dict(uniform=f.cpu()),
                   dict(logits=torch.zeros(1, 100, device=DEV).expand(4, 100)), dict(temperature=torch.ones(8, device=DEV)[::2])):
        with pytest.raises(ops.KernelError):
            ops.sample_filtered(**{**good, **change})
