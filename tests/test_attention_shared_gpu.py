"""ops.paged_attention_shared against the formula in 64 bits, over a cache in which everything that no row may see is NaN."""
import numpy as np
import pytest
import torch

from imparo_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Batch:
    """Rows in groups (rows, shared positions), own positions per row, their pages in any order.  extra rows belong to no group."""

    def __init__(self, groups, own, nh, nkv, hd, dtype, page=16, seed=0, extra=0, scale=None, q_size=1.5):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.hd, self.page, self.dtype = nh, nkv, hd, page, dtype
        rows = sum(n for n, _ in groups) + extra
        group_of = [g for g, (n, _) in enumerate(groups) for _ in range(n)] + [-1] * extra
        self.own = [int(own(r)) if callable(own) else own for r in range(rows)]
        lens = [(groups[g][1] if g >= 0 else 0) + self.own[r] for r, g in enumerate(group_of)]
        blocks = [-(-n // page) for n in lens]
        whole = [s // page for _, s in groups]
        self.n_pages = sum(whole) + sum(blocks) + 2
        pages = rng.permutation(self.n_pages)
        table = np.full((rows, max(max(blocks), 1) + 1), -1, dtype=np.int32)
        k = np.full((self.n_pages, page, nkv * hd), np.nan, dtype=np.float32)
        v = k.copy()
        at, self.first_of = 0, {}
        for r, g in enumerate(group_of):
            if g >= 0 and g not in self.first_of:
                self.first_of[g] = r
                table[r, :whole[g]] = pages[at:at + whole[g]]
                at += whole[g]
            n = whole[g] if g >= 0 else 0
            if n:
                table[r, :n] = table[self.first_of[g], :n]
            mine = max(0, blocks[r] - n)
            table[r, n:n + mine] = pages[at:at + mine]
            at += mine
            first = g < 0 or self.first_of[g] == r
            for pos in range(0 if first else groups[g][1], lens[r]):
                k[table[r, pos // page], pos % page] = rng.standard_normal(nkv * hd)
                v[table[r, pos // page], pos % page] = rng.standard_normal(nkv * hd)
            if not first and groups[g][1] % page and blocks[r] > n:            # a copy of the page the shared positions end in
                src, dst, part = table[self.first_of[g], n], table[r, n], groups[g][1] % page
                k[dst, :part], v[dst, :part] = k[src, :part], v[src, :part]
        dev = lambda x, t=torch.int32: torch.tensor(np.asarray(x), dtype=t, device=DEV)
        self.k, self.v = dev(k, dtype), dev(v, dtype)
        self.q = (torch.tensor(rng.standard_normal((rows, nh * hd)), device=DEV) * q_size).to(dtype)
        self.table, self.items = dev(table), dev(np.arange(rows))
        self.positions = dev([n - 1 for n in lens])
        self.group_start = dev(np.concatenate([[0], np.cumsum([n for n, _ in groups])]))
        self.shared = dev([s for _, s in groups])
        self.scale = 1 / np.sqrt(hd) if scale is None else scale
        self.most_shared, self.most_own = max(s for _, s in groups), max(self.own + [0])
        self.status = ops.new_status(DEV)

    def run(self, window=None, sinks=None, plan=None, q=None, out=None, check=True):
        q = self.q if q is None else q
        T = q.shape[0]
        plan = plan or ops.shared_prefix_plan(T, self.shared.numel(), self.nh, self.nkv, self.hd, self.dtype, self.most_shared, self.most_own)
        out = torch.full((T, self.nh * self.hd), float("nan"), dtype=self.dtype, device=DEV) if out is None else out
        scratch = [torch.full((n,), float("nan"), dtype=torch.float32, device=DEV) for n in (plan.acc_floats, plan.ml_floats)]
        ops.paged_attention_shared(q, self.k, self.v, self.positions, self.items, self.table, self.page, self.n_pages, self.group_start,
                                   self.shared, window, self.scale, out, *scratch, plan, self.nh, self.nkv, self.hd, self.status,
                                   sink_values=sinks)
        if check:
            ops.read_status(self.status)
        return out

    def plain(self, window=None, sinks=None):
        """(result, bound on the error of its parts) in 64 bits."""
        nh, nkv, hd, page = self.nh, self.nkv, self.hd, self.page
        q, k, v = (x.double().cpu().numpy() for x in (self.q, self.k, self.v))
        table, pos = self.table.cpu().numpy(), self.positions.cpu().numpy()
        items = self.items.cpu().numpy()
        out, bound = np.zeros((len(q), nh, hd)), np.zeros((len(q), nh, hd))
        eps = 2.0 ** -24
        for r in range(len(q)):
            lo = max(0, pos[r] + 1 - window) if window else 0
            at = np.arange(lo, pos[r] + 1)
            if not len(at):
                continue
            kk, vv = (x[table[items[r], at // page], at % page].reshape(-1, nkv, hd) for x in (k, v))
            for h in range(nh):
                key, qq = kk[:, h * nkv // nh], q[r].reshape(nh, hd)[h]
                s = key @ qq * self.scale
                # a 32-bit score is off by (head size + 2) roundings of its terms' sizes, the exponent's argument (in units of
                # log2 e) by three more of its own
                ds = (hd + 2) * eps * (np.abs(key) @ np.abs(qq)) * self.scale + 3 * eps * np.abs(s).max()
                top = s.max() if sinks is None else max(s.max(), float(sinks[h]))
                p = np.exp(s - top)
                total = p.sum() + (0 if sinks is None else np.exp(float(sinks[h]) - top))
                out[r, h] = p @ vv[:, h * nkv // nh] / total
                spread = np.abs(vv[:, h * nkv // nh]).T @ p / total
                # a weight's relative error: its score's, 2 ulp of the exponential, and the max's (cancels but for rounding); the sums
                # add one rounding per term at worst, tree or chain
                rel = 2 * ds.max() + (len(at) + 16) * eps
                # 16-bit: each weight is rounded once more (half a step: 2^-8) and so is the result
                bound[r, h] = rel * (spread + np.abs(out[r, h]))
                if self.dtype == torch.bfloat16:
                    bound[r, h] += 2.0 ** -8 * (spread + np.abs(out[r, h])) + 2.0 ** -16 * spread
        return out.reshape(len(q), -1), bound.reshape(len(q), -1)

    def check(self, **kw):
        got = self.run(**kw).double().cpu().numpy()
        want, bound = self.plain(**{k: v for k, v in kw.items() if k in ("window", "sinks")})
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) - bound).max()
        assert (np.abs(got - want) <= bound + 1e-30).all(), f"beyond the bound by {worst:.3e}"
        return got


TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [16, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (6, 2), (8, 2), (8, 1), (20, 1), (32, 1)])
def test_heads_and_sizes(dtype, hd, nh, nkv):
    Batch([(5, 70), (3, 33)], lambda r: 1 + 7 * r, nh, nkv, hd, dtype).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shared", [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 300, 1000, 2049])
def test_shared_lengths(dtype, hd, shared):
    Batch([(3, shared)], lambda r: 1 + 20 * r, 8, 2, hd, dtype, seed=shared).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("own", [1, 2, 63, 64, 65, 130, 700, 1500])
def test_own_lengths(dtype, hd, own):
    Batch([(2, 200)], lambda r: own + r, 8, 2, hd, dtype, seed=own).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 2, 16, 31, 32, 33, 63, 64, 65, 100, 140])
def test_rows_of_a_group(dtype, hd, rows):
    """Fewer rows than a tile of queries, exactly one, one more, several."""
    Batch([(rows, 333)], lambda r: 1 + r % 5, 4, 1, hd, dtype, seed=rows).check()


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("group", [33, 64, 100, 128, 130])
def test_many_heads_to_a_kv_head(dtype, hd, group):
    Batch([(3, 190), (2, 64)], lambda r: 1 + 40 * r, 2 * group, 2, hd, dtype, extra=1, seed=group).check()


@pytest.mark.parametrize("page", [48, 96, 192])
@pytest.mark.parametrize("window", [None, 150])
def test_page_sizes_that_are_no_power_of_two(page, window):
    Batch([(4, 500), (2, 199)], lambda r: 3 + 70 * r, 4, 2, 64, torch.bfloat16, page=page).check(window=window)


@pytest.mark.parametrize("page", [1, 5, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_page_sizes(dtype, hd, page):
    Batch([(4, 275), (2, 130)], lambda r: 3 + r, 4, 2, hd, dtype, page=page).check()


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 96)])
class TestRows:
    def test_groups_of_all_kinds(self, dtype, hd):
        """Empty groups, groups of one row, rows of no group, a group that shares nothing, a shared part of odd length."""
        Batch([(3, 401), (0, 64), (1, 150), (5, 0), (2, 16)], lambda r: 1 + 11 * r, 8, 2, hd, dtype, extra=3).check()

    def test_windows(self, dtype, hd):
        b = Batch([(4, 300), (3, 100)], lambda r: 1 + 30 * r, 4, 2, hd, dtype)
        for window in (1, 2, 40, 129, 200, 350, 10000):
            b.check(window=window)

    def test_sinks(self, dtype, hd):
        b = Batch([(4, 300)], lambda r: 1 + 3 * r, 8, 2, hd, dtype)
        b.check(sinks=torch.tensor([-50.0, -2.0, 0.0, 1.0, 3.0, 8.0, 30.0, 80.0], device=DEV))

    @pytest.mark.parametrize("rows", [6, 90])
    @pytest.mark.parametrize("most_own", [20, 2000])
    def test_sinks_of_minus_infinity_are_none(self, dtype, hd, rows, most_own):
        """exp(-inf) adds nothing: as without a sink, and zeros for a row that sees nothing."""
        b = Batch([(rows, 100)], 20, 4, 2, hd, dtype)
        b.positions[1] = -1
        plan = ops.shared_prefix_plan(rows, 1, 4, 2, hd, dtype, 100, most_own)
        want = b.run(plan=plan)
        some = torch.tensor([float("-inf"), 0.5, float("-inf"), -1.0], device=DEV)
        got = b.run(plan=plan, sinks=some).view(rows, 4, hd)
        assert not got[1].any() and torch.equal(got[:, ::2], want.view(rows, 4, hd)[:, ::2])
        assert torch.equal(b.run(plan=plan, sinks=torch.full((4,), float("-inf"), device=DEV)), want)

    def test_rows_without_a_position_and_rows_that_end_inside_the_shared_part(self, dtype, hd):
        b = Batch([(6, 260), (2, 40)], 9, 8, 2, hd, dtype, extra=1)
        pos = b.positions.clone()
        pos[1], pos[3], pos[4], pos[7], pos[8] = -1, 100, 259, 0, -1
        b.positions = pos
        got = b.check()
        assert not got[1].any() and not got[8].any()
        b.positions = torch.full_like(pos, -1)
        assert not b.check().any()

    def test_a_masked_row_beside_infinite_values(self, dtype, hd):
        """A row that ends before a position does not feel what lies there."""
        b = Batch([(3, 200)], 5, 4, 2, hd, dtype)
        b.positions[0] = 149
        want = b.run()[0].clone()
        b.v[b.table[0, 160 // 16], 3] = float("inf")
        b.k[b.table[0, 176 // 16], 2] = float("nan")
        assert torch.equal(b.run()[0], want)

    def test_queries_of_a_wider_buffer(self, dtype, hd):
        b = Batch([(5, 170)], 9, 4, 2, hd, dtype)
        wide = torch.full((5, b.nh * hd + 3 * hd), float("nan"), dtype=dtype, device=DEV)
        wide[:, hd:hd + b.nh * hd] = b.q
        assert torch.equal(b.run(q=wide[:, hd:hd + b.nh * hd]), b.run())
        odd = torch.full((5, b.nh * hd + 13), float("nan"), dtype=dtype, device=DEV)
        odd[:, 1:1 + b.nh * hd] = b.q
        b.q = odd[:, 1:1 + b.nh * hd]
        b.check()

    def test_large_scores(self, dtype, hd):
        """One key takes all the weight; the largest score comes last, first, in between."""
        b = Batch([(4, 500)], 40, 4, 2, hd, dtype, q_size=40.0)
        b.check()

    def test_a_plan_made_for_other_lengths(self, dtype, hd):
        b = Batch([(4, 700), (2, 90)], lambda r: 5 + 60 * r, 4, 2, hd, dtype)
        for shared, own in ((0, 0), (64, 1), (5000, 3000)):
            plan = ops.shared_prefix_plan(6, 2, 4, 2, hd, dtype, shared, own)
            b.check(plan=plan)

    def test_one_row_does_not_depend_on_its_neighbours(self, dtype, hd):
        b = Batch([(6, 300)], 21, 4, 2, hd, dtype)
        plan = ops.shared_prefix_plan(6, 1, 4, 2, hd, dtype, 300, 21)
        first = b.run(plan=plan)
        b.q[1:] = b.q[1:].flip(0)
        assert torch.equal(b.run(plan=plan)[0], first[0])
        assert torch.equal(b.run(plan=plan), b.run(plan=plan))

    def test_items_in_any_order(self, dtype, hd):
        b = Batch([(4, 200), (3, 64)], lambda r: 1 + r, 4, 2, hd, dtype)
        want = b.run()
        order = torch.tensor([5, 2, 6, 0, 3, 1, 4], device=DEV)
        table = torch.empty_like(b.table)
        table[order] = b.table
        b.table, b.items = table, order.int()
        assert torch.equal(b.run(), want)

    def test_bad_pages_and_items_are_reported(self, dtype, hd):
        for what in ("page", "unmapped", "item"):
            b = Batch([(4, 200)], 30, 4, 2, hd, dtype)
            if what == "item":
                b.items[2] = 99
            else:
                b.table[0 if what == "page" else 3, 3 if what == "page" else 13] = b.n_pages if what == "page" else -1
            b.run(check=False)
            with pytest.raises(ops.KernelError):
                ops.read_status(b.status)

    def test_positions_far_beyond_the_table_are_reported(self, dtype, hd):
        """At once, not after two thousand million keys; the other rows are as they were."""
        for which, window in ((slice(1, 2), None), (slice(0, 4), None), (slice(2, 3), 100)):
            b = Batch([(4, 200), (2, 50)], 30, 4, 2, hd, dtype)
            want = b.run(window=window)
            b.positions[which] = 0x7fffffff
            if which.stop == 4:
                b.shared[0] = 0x7fffffff
            got = b.run(window=window, check=False)
            with pytest.raises(ops.KernelError):
                ops.read_status(b.status)
            assert torch.equal(got[4:], want[4:])

    def test_a_group_of_rows_without_a_position_looks_nothing_up(self, dtype, hd):
        """All of its continuations have ended and their pages are gone, whatever its shared length still says."""
        b = Batch([(4, 200), (3, 150), (2, 64)], 30, 4, 2, hd, dtype)
        want = b.run()
        b.positions[4:7] = -1
        b.table[4:7] = -1
        for shared in (150, 0x7fffffff):
            b.shared[1] = shared
            got = b.run()
            assert not got[4:7].any() and torch.equal(got[:4], want[:4]) and torch.equal(got[7:], want[7:])

    def test_the_first_continuations_of_a_group_have_ended(self, dtype, hd):
        b = Batch([(1, 40), (40, 200), (2, 64)], 30, 4, 2, hd, dtype)
        plan = ops.shared_prefix_plan(43, 3, 4, 2, hd, dtype, 200, 30)
        b.positions[1:36] = -1
        want = b.run(plan=plan)
        b.table[1:36] = -1
        b.items[1:36] = 0
        got = b.run(plan=plan)
        assert torch.equal(got, want) and not got[1:36].any() and got[36:41].any(dim=1).all()

    def test_captured_and_replayed(self, dtype, hd):
        b = Batch([(4, 300), (2, 64)], lambda r: 9 + r, 4, 2, hd, dtype)
        plan = ops.shared_prefix_plan(6, 2, 4, 2, hd, dtype, 300, 20)
        out = torch.zeros(6, 4 * hd, dtype=dtype, device=DEV)
        acc, ml = torch.empty(plan.acc_floats, device=DEV), torch.empty(plan.ml_floats, device=DEV)
        run = lambda: ops.paged_attention_shared(b.q, b.k, b.v, b.positions, b.items, b.table, 16, b.n_pages, b.group_start, b.shared, None,
                                                 b.scale, out, acc, ml, plan, 4, 2, hd, b.status)
        run()
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            run()
        b.q.mul_(-0.5)
        b.positions.sub_(torch.tensor([0, 3, 1, 0, 4, 2], dtype=torch.int32, device=DEV))
        want = b.run(plan=plan)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(out, want)


def test_many_rows_and_long_prefix():
    """More key stretches than fill the chip once, several tiles of queries."""
    b = Batch([(70, 5000), (9, 3000)], lambda r: 1 + r % 50, 8, 2, 64, torch.bfloat16)
    b.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [90, 170])
class TestManyRows:
    """So many rows that a row's own keys are taken by one CTA for several kv heads, one or two to an SM."""

    @pytest.mark.parametrize("nh,nkv", [(2, 2), (6, 2), (16, 2), (6, 3), (33, 11)])
    def test_heads(self, hd, rows, nh, nkv):
        Batch([(rows, 100)], lambda r: 1 + 29 * r % 71, nh, nkv, hd, torch.bfloat16).check()

    @pytest.mark.parametrize("window", [None, 1, 150])
    def test_groups_of_all_kinds(self, hd, rows, window):
        b = Batch([(rows - 8, 333), (0, 5), (3, 0), (1, 70), (2, 48)], lambda r: 1 + 37 * r % 200, 8, 2, hd, torch.bfloat16, extra=2)
        b.positions[3] = b.positions[rows - 1] = -1
        b.positions[7] = b.positions[7] // 2 if window is None else b.positions[7]
        got = b.check(window=window)
        assert not got[3].any() and not got[rows - 1].any()
        b.check(window=window, sinks=torch.tensor([-50.0, -2.0, 0.0, 1.0, 3.0, 8.0, 30.0, 80.0], device=DEV))

    @pytest.mark.parametrize("page", [1, 5, 64])
    def test_page_sizes(self, hd, rows, page):
        Batch([(rows - 5, 130), (5, 64)], lambda r: 1 + r % 50, 4, 2, hd, torch.bfloat16, page=page).check()

    def test_long_rows_among_short_ones(self, hd, rows):
        """More own keys than are looked up at once, just as many, one more."""
        b = Batch([(rows, 40)], lambda r: {0: 1024, 5: 1025, 9: 1023, 40: 2100, 80: 1040}.get(r, 1 + r % 20), 4, 2, hd, torch.bfloat16)
        plan = ops.shared_prefix_plan(rows, 1, 4, 2, hd, torch.bfloat16, 40, 100)
        assert plan.n_own == 1
        b.check(plan=plan)

    def test_a_row_does_not_feel_its_neighbours_or_what_it_may_not_see(self, hd, rows):
        b = Batch([(rows, 100)], 37, 8, 2, hd, torch.bfloat16)
        b.positions[2] = 119                                       # of 136
        plan = ops.shared_prefix_plan(rows, 1, 8, 2, hd, torch.bfloat16, 100, 37)
        want = b.run(plan=plan)
        b.v[b.table[2, 7], 8:] = float("inf")                      # positions 120 to 127
        b.k[b.table[2, 8]] = float("nan")
        b.q[3:] = b.q[3:].flip(0)
        got = b.run(plan=plan)
        assert torch.equal(got[:3], want[:3]) and torch.equal(b.run(plan=plan), got)

    @pytest.mark.parametrize("what", ["page", "unmapped", "item", "far"])
    def test_what_is_wrong_is_reported(self, hd, rows, what):
        b = Batch([(rows, 64)], 30, 4, 2, hd, torch.bfloat16)
        want = b.run()
        if what == "item":
            b.items[2] = 9999
        elif what == "far":
            b.positions[2] = 0x7fffffff
        else:
            b.table[2, 5] = b.n_pages if what == "page" else -1
        got = b.run(check=False)
        with pytest.raises(ops.KernelError):
            ops.read_status(b.status)
        assert torch.equal(got[3:], want[3:])


@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("dtype,hd,rows,most_own", [(torch.float32, 64, 4, 40), (torch.float32, 64, 4, 2000), (torch.bfloat16, 96, 4, 40),
                                                    (torch.bfloat16, 64, 4, 40), (torch.bfloat16, 64, 4, 2000), (torch.bfloat16, 64, 90, 40),
                                                    (torch.bfloat16, 128, 4, 40), (torch.bfloat16, 128, 4, 2000), (torch.bfloat16, 128, 90, 40)])
class TestNoNumbers:
    """A score that is no number or infinite, in whichever stretch of whichever kernel: who sees it has no result, the others theirs."""

    def setup(self, where, dtype, hd, rows, most_own):
        b = Batch([(rows, 200)], 40, 4, 2, hd, dtype)
        plan = ops.shared_prefix_plan(rows, 1, 4, 2, hd, dtype, 200, most_own)
        pos = 77 if where == "shared" else 215                     # an own one is row 1's alone
        place = b.k[b.table[1, pos // 16], pos % 16]
        sees = torch.ones(rows, dtype=torch.bool, device=DEV) if where == "shared" else torch.arange(rows, device=DEV) == 1
        return b, plan, place, sees

    def test_a_key_that_is_no_number(self, where, dtype, hd, rows, most_own):
        b, plan, place, sees = self.setup(where, dtype, hd, rows, most_own)
        want = b.run(plan=plan).view(rows, 4, hd)
        place[3] = float("nan")                                    # of the first kv head: query heads 0 and 1
        got = b.run(plan=plan).view(rows, 4, hd)
        assert got[sees, :2].isnan().all()
        assert torch.equal(got[sees, 2:], want[sees, 2:]) and torch.equal(got[~sees], want[~sees])

    def test_an_infinite_score(self, where, dtype, hd, rows, most_own):
        """Above all others: none has a finite share.  Below all: a share of 0, as that of a very low score."""
        b, plan, place, sees = self.setup(where, dtype, hd, rows, most_own)
        q = b.q.view(rows, 4, hd)
        q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
        place[0] = 1e30
        want = b.run(plan=plan).view(rows, 4, hd)
        assert want.isfinite().all()
        place[0] = float("inf")
        got = b.run(plan=plan).view(rows, 4, hd)
        assert got[sees, 0].isnan().all()
        assert torch.equal(got[sees, 1:], want[sees, 1:]) and torch.equal(got[~sees], want[~sees])

    def test_a_query_that_is_no_number(self, where, dtype, hd, rows, most_own):
        b, plan, _, _ = self.setup(where, dtype, hd, rows, most_own)
        sinks = torch.tensor([0.5, -1.0, 2.0, 0.0], device=DEV) if where == "own" else None
        want = b.run(plan=plan, sinks=sinks).view(rows, 4, hd)
        b.q[2, hd + 5] = float("nan")                              # row 2, head 1
        got = b.run(plan=plan, sinks=sinks).view(rows, 4, hd)
        assert got[2, 1].isnan().all()
        want[2, 1] = got[2, 1] = 0
        assert torch.equal(got, want)


def test_no_rows():
    b = Batch([(2, 30)], 2, 4, 2, 64, torch.bfloat16)
    plan = ops.shared_prefix_plan(1, 1, 4, 2, 64, torch.bfloat16, 30, 2)
    b.run(q=b.q[:0], plan=plan)


def test_refusals():
    b = Batch([(3, 100)], 4, 4, 2, 64, torch.bfloat16)
    plan = ops.shared_prefix_plan(3, 1, 4, 2, 64, torch.bfloat16, 100, 4)
    acc, ml = torch.empty(plan.acc_floats, device=DEV), torch.empty(plan.ml_floats, device=DEV)
    out = torch.empty_like(b.q)
    names = ("q", "k_cache", "v_cache", "positions", "item_of_token", "table", "page_size", "n_pages", "group_start", "shared_len", "window",
             "scale", "out", "part_acc", "part_ml", "plan", "nh", "nkv", "hd", "status")
    good = dict(zip(names, (b.q, b.k, b.v, b.positions, b.items, b.table, 16, b.n_pages, b.group_start, b.shared, None, b.scale, out, acc, ml,
                            plan, 4, 2, 64, b.status)))
    ops.paged_attention_shared(**good)
    for change in (dict(q=b.q.float()), dict(q=b.q.half(), out=out.half(), k_cache=b.k.half(), v_cache=b.v.half()), dict(k_cache=b.k.float()),
                   dict(positions=b.positions.long()), dict(positions=b.positions[:2]), dict(table=b.table.long()), dict(table=b.table[0]),
                   dict(group_start=b.group_start[:1]), dict(shared_len=b.shared.float()), dict(out=out[:2]), dict(part_acc=acc[:-1]),
                   dict(part_ml=ml[:-1]), dict(n_pages=b.n_pages + 1), dict(nh=3), dict(hd=63), dict(nh=16, nkv=8, hd=16, q=b.q[:, :256].float()),
                   dict(status=b.status.cpu()), dict(sink_values=torch.zeros(3, device=DEV)), dict(window=-1),
                   dict(plan=plan._replace(n_shared=4000)), dict(plan=plan._replace(n_own=0)), dict(item_of_token=b.items.cpu()),
                   dict(page_size=0), dict(v_cache=b.v[:-1])):
        with pytest.raises(ops.KernelError):
            ops.paged_attention_shared(**{**good, **change})
