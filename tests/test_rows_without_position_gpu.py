"""Rows of position -1 (no request's: what ops.step_tables leaves behind a step's tokens) through every kernel that writes to the paged cache:
they write nothing there, they are not reported, and the other rows are as they are without them."""
import pytest
import torch

from imparo_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE, PAGES, PAD = 16, 80, 5
F32, BF16 = torch.float32, torch.bfloat16


def arena(width, dtype):
    """A cache with a page's worth of memory around it that nobody may write to."""
    whole = torch.full((PAGES + 2, PAGE, width), -77.0, dtype=dtype, device=DEV)
    return whole, whole[1:-1]


def run(call, rows, dtype, widths):
    """call(rows of the batch, positions, items, table, caches, status) -> tensors of a row each; with and without rows of no position."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(rows)
    pages = torch.randperm(PAGES - 1, generator=gen, device=DEV).int() + 1
    table = torch.cat([torch.zeros_like(pages[:1]), pages]).view(8, PAGES // 8)        # the first item's first page: the arena's first one
    items = torch.arange(rows, device=DEV, dtype=torch.int32) % 8
    positions = torch.arange(rows, device=DEV, dtype=torch.int32) // 8 + 3
    results = []
    for pad in (0, PAD):
        no = torch.full((pad,), -1, dtype=torch.int32, device=DEV)
        status = ops.new_status(DEV)
        arenas = [arena(w, dtype) for w in widths]
        out = call(rows + pad, torch.cat([positions, no]), torch.cat([items, no * 0]), table, [a[1] for a in arenas], status)
        ops.read_status(status)
        results.append([x[:rows] for x in out] + [a[0] for a in arenas])
    for got, want in zip(results[1], results[0]):
        assert torch.equal(got, want)
    return results[0]


def rand(seed, *shape, dtype=F32):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=gen).to(dtype)


def inv(n_rot):
    return 10000.0 ** (-torch.arange(n_rot // 2, device=DEV, dtype=F32) * 2 / n_rot)


@pytest.mark.parametrize("rows", [9, 300, 600])
@pytest.mark.parametrize("dtype,hd,n_rot,aligned", [(F32, 64, 64, True), (F32, 48, 16, True), (BF16, 64, 64, True), (BF16, 128, 128, True),
                                                    (BF16, 256, 256, True), (BF16, 64, 64, False), (BF16, 96, 64, True)])
def test_qk_norm_rope_store(rows, dtype, hd, n_rot, aligned):
    nh, nkv = 4, 2
    weight = rand(2, hd + 1).abs()
    weight = weight[:hd] if aligned else weight[1:]

    def call(T, positions, items, table, caches, status):
        qkv = rand(1, 700, (nh + 2 * nkv) * hd, dtype=dtype)[:T].contiguous()
        q = torch.zeros(T, nh * hd, dtype=dtype, device=DEV)
        ops.qk_norm_rope_store(qkv, positions, items, weight, weight, inv(n_rot), n_rot, 1e-6, q, *caches, table, PAGE, PAGES, nh, nkv, hd, status)
        return [q]
    assert (run(call, rows, dtype, [nkv * hd] * 2)[1] != -77).any()


@pytest.mark.parametrize("rows", [9, 300])
@pytest.mark.parametrize("dtype,interleaved", [(F32, True), (F32, False), (BF16, True), (BF16, False)])
def test_qkv_rotate_store(rows, dtype, interleaved):
    nh, nkv, hd, vd = 3, 1, 24, 40

    def call(T, positions, items, table, caches, status):
        qkv = rand(1, 400, nh * hd + nkv * (hd + vd), dtype=dtype)[:T].contiguous()
        q = torch.zeros(T, nh * hd, dtype=dtype, device=DEV)
        ops.qkv_rotate_store(qkv, positions, items, inv(8), 8, interleaved, 1.0, q, *caches, table, PAGE, PAGES, nh, nkv, hd, vd, status)
        return [q]
    run(call, rows, dtype, [nkv * hd, nkv * vd])


@pytest.mark.parametrize("rows", [9, 300])
@pytest.mark.parametrize("dtype,hd", [(F32, 24), (F32, 25), (BF16, 24), (BF16, 64)])
def test_qkv_norm_rotate_store(rows, dtype, hd):
    nh, nkv, vd = 3, 2, hd

    def call(T, positions, items, table, caches, status):
        qkv = rand(1, 400, nh * hd + nkv * (hd + vd), dtype=dtype)[:T].contiguous()
        q, w = torch.zeros(T, nh * hd, dtype=dtype, device=DEV), torch.ones(hd, device=DEV)
        ops.qkv_norm_rotate_store(qkv, positions, items, w, w, 1e-6, inv(16), 16, q, *caches, table, PAGE, PAGES, nh, nkv, hd, vd, status)
        return [q]
    run(call, rows, dtype, [nkv * hd, nkv * vd])


@pytest.mark.parametrize("rows", [9, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("unit_eps", [None, 1e-6])
def test_qkv_prepare_store(rows, dtype, unit_eps):
    nh, nkv, hd, vd = 3, 2, 32, 32

    def call(T, positions, items, table, caches, status):
        qkv = rand(1, 400, nh * hd + nkv * (hd + vd))[:T].contiguous()
        q = torch.zeros(T, nh * hd, dtype=dtype, device=DEV)
        ops.qkv_prepare_store(qkv, None, positions, items, inv(16), 16, unit_eps, None, None, None, q, *caches, table, PAGE, PAGES, nh, nkv, hd, vd,
                              status)
        return [q]
    run(call, rows, dtype, [nkv * hd, nkv * vd])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_latent_stores(dtype):
    rank, q_rank, heads, dim, rot = 64, 48, 3, 32, 16

    def plain(T, positions, items, table, caches, status):
        proj = rand(1, 40, q_rank + rank)[:T].contiguous()
        q = torch.zeros(T, q_rank, dtype=dtype, device=DEV)
        ops.latent_norm_store(proj, 0, q_rank, q_rank, rank, torch.ones(q_rank, device=DEV), torch.ones(rank, device=DEV), 1e-6, positions, items, q,
                              caches[0], table, PAGE, PAGES, status)
        return [q]

    def turned(T, positions, items, table, caches, status):
        proj = rand(1, 40, heads * (dim + rot) + rank + rot)[:T].contiguous()
        q, lat = torch.zeros(T, heads * dim, dtype=dtype, device=DEV), torch.zeros(T, heads * (rank + rot), dtype=dtype, device=DEV)
        ops.latent_rot_store(proj, heads, dim, rot, rank, torch.ones(rank, device=DEV), 1e-6, inv(rot), rot, positions, items, q, lat, caches[0],
                             table, PAGE, PAGES, status)
        return [q, lat.view(T, heads, -1)[:, :, rank:]]
    run(plain, 9, dtype, [rank])
    run(turned, 9, dtype, [rank + rot])


def test_a_page_that_is_missing_is_still_reported():
    table = torch.full((1, 2), -1, dtype=torch.int32, device=DEV)
    zero, status = torch.zeros(1, dtype=torch.int32, device=DEV), ops.new_status(DEV)
    q, (k, v) = torch.zeros(1, 128, device=DEV), (arena(64, F32)[1] for _ in range(2))
    ops.qk_norm_rope_store(rand(1, 1, 256), zero, zero, None, None, inv(64), 64, 1e-6, q, k, v, table, PAGE, PAGES, 2, 1, 64, status)
    with pytest.raises(ops.KernelError):
        ops.read_status(status)


@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("which,dtype", [("any head", F32), ("any head", BF16), ("split", F32), ("split", BF16), ("general", F32), ("general", BF16),
                                         ("shared heads", BF16), ("sigmoid", BF16)])
def test_attention_of_rows_without_a_position_is_zero(which, dtype, window):
    nh, nkv, hd, rows = 4, 2, 64, 9

    def call(T, positions, items, table, caches, status):
        q, out = rand(1, 40, nh * hd, dtype=dtype)[:T].contiguous(), torch.full((T, nh * hd), 3.0, dtype=dtype, device=DEV)
        caches = [rand(5 + i, PAGES, PAGE, nkv * hd, dtype=dtype) for i in range(2)]
        chunk, n_splits = ops.split_plan(rows, nkv, table.shape[1] * PAGE)
        acc, ml = torch.empty(T * nh * n_splits * hd, device=DEV), torch.empty(T * nh * n_splits * 2, device=DEV)
        head = (q, *caches, positions, items, table, PAGE, PAGES, window)
        if which == "any head":
            ops.paged_attention(*head, 0.125, out, nh, nkv, hd, status)
        elif which == "split":
            assert ops.paged_attention_split(*head, 0.125, out, acc, ml, chunk, n_splits, nh, nkv, hd, status)
        elif which == "general":
            ops.attention_any(*head, 0.125, True, out, nh, nkv, hd, hd, status)
        elif which == "shared heads":
            assert ops.paged_attention_split_shared(*head, 0.125, out, acc, ml, chunk, n_splits, nh, nkv, hd, status)
        else:
            assert ops.attention_sigmoid_split(*head, None, 0.125, torch.zeros(nh, device=DEV), out, acc, ml, chunk, n_splits, nh, nkv, hd, hd, status)
        assert not out[rows:].any() and out[:rows].any(dim=1).all()
        return [out]
    run(call, rows, dtype, [8])
