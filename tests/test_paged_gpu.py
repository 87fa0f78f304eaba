"""Paged K/V cache operators against their 64-bit forms (tests/paged_ref.py)."""

import math
import subprocess
import sys

import pytest
import torch

from hspmn_b200 import _native as N
from hspmn_b200 import ops
from tests import paged_ref as ref
from tests.conftest import PKG, REPO

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# paged_slots_
# ---------------------------------------------------------------------------


def run_slots(seq, new, page, n, free=None, width=None, view=False):
    R = len(seq)
    g = torch.Generator().manual_seed(R + page)
    held = [-(-max(c, 0) // page) for c in seq]
    want = [-(-(max(c, 0) + max(m, 0)) // page) for c, m in zip(seq, new)]
    width = max(want + [1]) + 1 if width is None else width
    pages = torch.randperm(sum(want) + 7, generator=g).tolist()
    rows, at = [], 0
    for h in held:
        rows.append((pages[at:at + h] + [-5] * width)[:width])
        at += h
    free = pages[at:] if free is None else pages[at:at + free]
    table = torch.full((R, 2 * width + 3), -9, dtype=torch.int32, device=DEV)
    if R:
        table[:, 1:1 + width] = i32(rows)
    t = table[:, 1:1 + width] if view else table[:, 1:1 + width].contiguous()
    got = ops.paged_slots_(t, i32(seq), i32(new), i32(free), page, n)
    want = ref.slots_ref(rows, seq, new, free, page, n)
    assert t.tolist() == want[0]
    for name, a, b in zip(("cu", "kv_lens", "positions", "slots"), got, want[1:5]):
        assert a.tolist() == b, name
    assert got[4].tolist() == [want[5]]
    if view:  # the columns beside the view are left as they were
        assert (table[:, 0] == -9).all() and (table[:, 1 + width:] == -9).all()
    return got


@pytest.mark.parametrize("page", [8, 16, 64, 4096])
@pytest.mark.parametrize("seq,new,pad", [
    ([0], [1], 0), ([0], [0], 3), ([5], [0], 0), ([15, 16, 17, 0, 63], [1, 1, 1, 1, 1], 0),
    ([0, 0, 0], [0, 700, 0], 5), ([4095, 4096, 1, 8191], [1, 1, 9000, 2], 1), ([7] * 300, [3] * 300, 0)])
def test_slots(page, seq, new, pad):
    run_slots(seq, new, page, sum(new) + pad, view=pad % 2 == 1)
    assert ops.device_errors() == 0


@pytest.mark.parametrize("R", [255, 256, 257, 1000, 8192])
def test_slots_many_requests(R):
    g = torch.Generator().manual_seed(R)
    seq = torch.randint(0, 200, (R,), generator=g).tolist()
    new = torch.randint(0, 40, (R,), generator=g).tolist()
    run_slots(seq, new, 16, sum(new) + 11)
    assert ops.device_errors() == 0


def test_slots_in_a_fresh_process():
    """From few requests to many in a process of its own: what one call asks of the runtime (more shared memory than
    a kernel gets by default) must not be what a smaller one needs."""
    code = ("import sys; sys.path[:0] = [%r, %r]\n"
            "from tests.test_paged_gpu import ops, run_slots\n"
            "for R in (1, 5800, 6000, 6014, 6015, 6016, 6017, 6080, 6134, 6135, 6136, 6143, 6144, 6145, 8191, 8192):\n"
            "    run_slots([15] * R, [1 + (R & 1)] * R, 16, (1 + (R & 1)) * R)\n"
            "    assert ops.device_errors() == 0\n" % (PKG, REPO))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_slots_empty_batch():
    run_slots([], [], 16, 0)
    run_slots([], [], 16, 4)
    assert ops.device_errors() == 0


def test_slots_flags_what_does_not_fit():
    run_slots([10, 0, 30], [20, 40, 5], 8, 65, free=4)  # the free list ends
    assert ops.device_errors() == N.DEVERR_PAGE
    run_slots([10, 0], [20, 40], 8, 60, width=4)  # the table is too narrow
    assert ops.device_errors() == N.DEVERR_POSITION
    run_slots([10, 0], [20, 40], 8, 33)  # more tokens than places
    assert ops.device_errors() == N.DEVERR_POSITION
    run_slots([-3, 4], [2, -7], 8, 4)  # negative lengths count as zero
    assert ops.device_errors() == N.DEVERR_POSITION
    t = torch.zeros((3, 4), dtype=torch.int32, device=DEV)
    big = 2 ** 31 - 1
    got = ops.paged_slots_(t, i32([big, 0, big]), i32([big, big, big]), i32([1, 2]), 8, 40)
    assert got[1].tolist() == [big] * 3 and got[3].max().item() < 3 * 8
    assert ops.device_errors() == N.DEVERR_POSITION | N.DEVERR_PAGE


def test_slots_flags_tokens_in_a_held_page_that_is_missing():
    """A request whose last page was never had (a step before found the free list at its end): its new tokens have no
    slot, and that is said; full pages that no new token goes to are not looked at."""
    table, free = i32([[4, -1, -1], [-1, 2, -1], [-7, 6, 7]]), i32([9])
    got = ops.paged_slots_(table, i32([12, 16, 20]), i32([3, 1, 0]), free, 8, 5)
    assert got[2].tolist() == [12, 13, 14, 16, -1] and got[3].tolist() == [-1, -1, -1, 9 * 8, -1]
    assert ops.device_errors() == N.DEVERR_PAGE
    got = ops.paged_slots_(i32([[-1, 2, -1], [-7, 6, 7]]), i32([15, 20]), i32([1, 0]), free, 8, 1)
    assert got[3].tolist() == [23] and ops.device_errors() == 0


# ---------------------------------------------------------------------------
# rope_paged_write_
# ---------------------------------------------------------------------------


def tables(L, hd, dtype, gen):
    ang = torch.rand((L, hd), generator=gen, dtype=torch.float64) * 6.28
    return ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tab", ["same", "f32", None])
@pytest.mark.parametrize("n,Hkv,hd,page,joint", [(1, 4, 128, 64, False), (61, 4, 64, 16, True), (130, 3, 48, 8, True),
                                                 (33, 16, 16, 32, False), (700, 1, 256, 128, True)])
def test_write(dtype, tab, n, Hkv, hd, page, joint):
    g = torch.Generator().manual_seed(n + hd)
    pages, L = -(-n // page) + 3, 2 * n + 5
    kv = torch.randn((pages, 2, page, Hkv, hd), generator=g).to(dtype).to(DEV)
    kc, vc = (kv[:, 0], kv[:, 1]) if joint else (kv[:, 0].contiguous(), kv[:, 1].contiguous())
    k0, v0 = kc.clone(), vc.clone()
    k = torch.randn((n, Hkv, hd), generator=g).to(dtype).to(DEV)
    v = torch.randn((n, Hkv, hd), generator=g).to(dtype).to(DEV)
    pos = torch.randint(0, L, (n,), generator=g).to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:n].to(DEV)
    slots[n // 2] = -1  # padding
    cos, sin = (None, None) if tab is None else tables(L, hd, dtype if tab == "same" else torch.float32, g)
    ops.rope_paged_write_(k, v, cos, sin, pos, slots, kc, vc)
    live = slots >= 0
    page_i, off = slots[live] // page, slots[live] % page
    assert torch.equal(vc[page_i, off], v[live])
    got = kc[page_i, off].double()
    if tab is None:
        assert torch.equal(got, k[live].double())
    else:
        want, size = ref.rope_ref(k[live], cos, sin, pos[live])
        # one rounding to the type, and three float32 operations before it
        u = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert ((got - want).abs() <= u * want.abs() * (1 + 1e-6) + 3 * 2.0 ** -24 * size + tiny).all()
    v0[page_i, off] = v[live]
    k0[page_i, off] = kc[page_i, off]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # nothing else was touched
    assert ops.device_errors() == 0


def test_write_takes_views_and_block_tables():
    """K and V as halves of one projection, tables as RotaryEmbedding keeps them."""
    from hspmn_b200 import RotaryEmbedding
    n, Hkv, hd, page = 37, 4, 64, 16
    kv = torch.randn(n, 2 * Hkv * hd, dtype=torch.bfloat16, device=DEV)
    k, v = kv[:, :Hkv * hd].view(n, Hkv, hd), kv[:, Hkv * hd:].view(n, Hkv, hd)
    rope = RotaryEmbedding(hd, 64).to(DEV)
    cos, sin = rope.cached_cos, rope.cached_sin  # float32 [1,1,L,hd]
    kc, vc = (torch.zeros((4, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pos, slots = torch.arange(n, device=DEV), torch.arange(n, device=DEV) + 3
    ops.rope_paged_write_(k, v, cos, sin, pos, slots, kc, vc)
    want, _ = ref.rope_ref(k, cos[0, 0], sin[0, 0], pos)
    got = kc.view(-1, Hkv, hd)[3:3 + n]
    assert torch.allclose(got.double(), want, rtol=2.0 ** -8, atol=2.0 ** -20)
    assert torch.equal(vc.view(-1, Hkv, hd)[3:3 + n], v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_write_takes_tables_of_any_layout(dtype):
    """Tables whose base or rows do not lie on 16 bytes, whose columns or rows are spread, of one row."""
    L, Hkv, hd, page = 9, 2, 64, 8
    g = torch.Generator().manual_seed(45)
    k = torch.randn((L, Hkv, hd), generator=g).to(torch.bfloat16).to(DEV)
    at = torch.arange(L, device=DEV)
    cos, sin = tables(L, hd, dtype, g)

    def write(cos, sin, rows=L):
        kc, vc = (torch.zeros((2, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ops.rope_paged_write_(k, k, cos, sin, at.clamp(max=rows - 1), at, kc, vc)
        return kc

    def shifted(t):
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    def odd_rows(t):
        return torch.zeros((L, hd + 1), dtype=t.dtype, device=DEV)[:, :hd].copy_(t)

    def columns_apart(t):
        return t.t().contiguous().t()

    want = write(cos, sin)
    for other in (shifted, odd_rows, columns_apart, lambda t: t[None, None], lambda t: odd_rows(t)[None, None]):
        assert torch.equal(write(other(cos), other(sin)), want)
        assert torch.equal(write(other(cos), sin), want) and torch.equal(write(cos, other(sin)), want)
    one = write(cos[:1].contiguous(), sin[:1].contiguous(), 1)
    for other in (lambda t: t[:1], lambda t: t[:1].as_strided((1, hd), (1, 1)), lambda t: t[:1].as_strided((1, hd), (0, 1)),
                  lambda t: t[0]):
        if other(cos).dim() == 1:
            with pytest.raises(ValueError):
                write(other(cos), other(sin), 1)
        else:
            assert torch.equal(write(other(cos), other(sin), 1), one)
    assert torch.equal(write(cos[:1].expand(L, hd), sin[:1].expand(L, hd)), one)
    assert ops.device_errors() == 0


def test_write_flags_bad_slots_and_positions():
    Hkv, hd, page = 2, 32, 8
    kc, vc = (torch.zeros((2, page, Hkv, hd), dtype=torch.float16, device=DEV) for _ in range(2))
    k = torch.ones((3, Hkv, hd), dtype=torch.float16, device=DEV)
    cos = torch.ones((4, hd), dtype=torch.float16, device=DEV)
    ops.rope_paged_write_(k, k, cos, cos, torch.tensor([0, 1, 2], device=DEV), torch.tensor([16, 5, 1 << 40], device=DEV),
                          kc, vc)
    assert ops.device_errors() == N.DEVERR_PAGE
    assert vc.view(16, -1).sum(1).nonzero().flatten().tolist() == [5]
    ops.rope_paged_write_(k, k, cos, cos, torch.tensor([4, 3, -1], device=DEV), torch.tensor([0, 6, 2], device=DEV), kc, vc)
    assert ops.device_errors() == N.DEVERR_POSITION
    assert vc.view(16, -1).sum(1).nonzero().flatten().tolist() == [5, 6]
    # without tables the positions are not read
    ops.rope_paged_write_(k, k, None, None, torch.tensor([9, 9, -9], device=DEV), torch.tensor([0, 1, 2], device=DEV), kc, vc)
    assert ops.device_errors() == 0 and vc.view(16, -1).sum(1).nonzero().flatten().tolist() == [0, 1, 2, 5, 6]


# ---------------------------------------------------------------------------
# sqdk_paged_fwd
# ---------------------------------------------------------------------------


def batch(kv_lens, positions, H, Hkv, hd, dtype, page, seed, joint=False, tail=0, fill=None):
    """``positions``: for each request its query positions."""
    g = torch.Generator().manual_seed(seed)
    kc, vc, table = ref.make_cache(kv_lens, page, Hkv, hd, dtype, g, DEV, joint, fill=fill)
    cu = [0]
    for ps in positions:
        cu.append(cu[-1] + len(ps))
    flat = [p for ps in positions for p in ps] + [0] * tail
    q = torch.randn((len(flat), H, hd), generator=g).to(dtype).to(DEV)
    return q, kc, vc, table, kv_lens, cu, torch.tensor(flat, dtype=torch.int64, device=DEV)


def attend(q, kc, vc, table, kv_lens, cu, pos, scale=None, max_q=0):
    return ops.sqdk_paged_fwd(q, kc, vc, table, i32(kv_lens), i32(cu), pos,
                              q.shape[-1] ** -0.5 if scale is None else scale, max_q)


def check(args, scale=None, max_qs=(0,)):
    q = args[0]
    want, tol = ref.attend_ref(*args, q.shape[-1] ** -0.5 if scale is None else scale)
    for max_q in max_qs:
        o = attend(*args, scale=scale, max_q=max_q)
        assert o.dtype == q.dtype and o.shape == q.shape and o.is_contiguous()
        err = (o.double() - want).abs()
        assert (err <= tol).all(), (max_q, err.max().item(), (err - tol).max().item())


HEADS = [(16, 4, 128), (16, 16, 64), (12, 4, 64), (6, 2, 96), (8, 1, 128), (4, 4, 8), (32, 1, 48), (128, 1, 64),
         (16, 2, 120)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,hd", HEADS)
def test_decode_heads(dtype, H, Hkv, hd):
    lens = [1, 7, 8, 63, 64, 65, 200]
    check(batch(lens, [[n - 1] for n in lens], H, Hkv, hd, dtype, 16, seed=H + hd, joint=hd == 64), max_qs=(0, 1))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("joint", [False, True])
def test_decode_pages(page, joint):
    lens = [1500, 3, page, page + 1, 2 * page - 1, 900]
    check(batch(lens, [[n - 1] for n in lens], 16, 4, 128, torch.bfloat16, page, seed=page, joint=joint), max_qs=(0, 1))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("R,n", [(1, 1), (1, 64), (1, 65), (1, 5000), (2, 20000), (300, 40), (40, 700)])
def test_decode_batches(R, n):
    """From fewer units than CTAs to many a CTA: items whole, cut once and cut often."""
    lens = [max(1, n - 13 * (r % 5)) for r in range(R)]
    check(batch(lens, [[m - 1] for m in lens], 8, 2, 64, torch.bfloat16, 16, seed=R + n), max_qs=(1,))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,hd", [(16, 4, 128), (12, 4, 64), (6, 2, 96), (4, 4, 64), (32, 1, 128), (40, 2, 16)])
def test_chunks(dtype, H, Hkv, hd):
    """Whole prompts, chunks behind cached tokens, selected rows, short runs and single tokens in one batch."""
    lens = [150, 331, 64, 40, 257, 500]
    positions = [list(range(150)), list(range(200, 331)), list(range(0, 64, 5)), [39], [254, 255, 256],
                 list(range(3, 500, 7))]
    check(batch(lens, positions, H, Hkv, hd, dtype, 16, seed=hd, joint=True), max_qs=(0, 150, 1))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("page", [8, 16, 32, 64, 256])
def test_chunk_pages(page):
    lens = [300, 77]
    check(batch(lens, [list(range(100, 300)), list(range(77))], 8, 2, 128, torch.bfloat16, page, seed=page),
          max_qs=(200,))
    assert ops.device_errors() == 0


def test_positions_in_any_order_and_repeated():
    lens = [200, 90]
    g = torch.Generator().manual_seed(5)
    positions = [torch.randperm(200, generator=g)[:77].tolist() + [13, 13, 13], [89, 0, 44, 44]]
    check(batch(lens, positions, 8, 2, 64, torch.bfloat16, 32, seed=1), max_qs=(0, 80))
    assert ops.device_errors() == 0


def test_rows_that_see_nothing_are_zero():
    lens = [0, 100, 70, 0, 64]
    positions = [[0], [-1, 5, 99, -7], list(range(70)), [], [63]]
    args = batch(lens, positions, 8, 2, 64, torch.bfloat16, 16, seed=2, tail=21)
    check(args, max_qs=(0, 70, 1))
    o = attend(*args)
    cu = args[5]
    assert not o[0].any() and not o[cu[1]].any() and not o[cu[1] + 3].any() and not o[cu[-1]:].any()
    assert ops.device_errors() == N.DEVERR_POSITION  # position 0 of a request with nothing cached
    none = attend(*batch([], [], 8, 2, 64, torch.bfloat16, 16, seed=2, tail=3))
    assert none.shape[0] == 3 and not none.any()
    assert attend(*batch([4], [[]], 8, 2, 64, torch.bfloat16, 16, seed=2)).shape == (0, 8, 64)
    assert ops.device_errors() == 0


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("page", [16, 64])
def test_what_lies_behind_the_last_token_does_not_count(fill, page):
    lens = [1, 50, 64, 65, 130, 300]
    positions = [[0], [49], [63], [64], list(range(100, 130)), list(range(60, 300))]
    check(batch(lens, positions, 16, 4, 64, torch.bfloat16, page, seed=3, fill=fill), max_qs=(0, 240))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_value_reaches_only_the_rows_that_see_its_key(bad, dtype):
    lens = [200, 40]
    args = batch(lens, [list(range(200)), [36, 37, 38, 39]], 8, 2, 64, dtype, 16, seed=4)
    q, kc, vc, table, _, cu, pos = args
    for r, p in ((0, 77), (0, 150), (1, 38)):
        vc[table[r, p // 16].item(), p % 16, 0, 5] = bad
        kc[table[r, p // 16].item(), p % 16, 1, 9] = bad
    want, tol = ref.attend_ref(*args, 0.125)
    for max_q in (0, 200):
        o = attend(*args, scale=0.125, max_q=max_q).double()
        assert torch.equal(o.isnan(), want.isnan())
        assert torch.equal(o[o.isinf()], want[o.isinf()]) and torch.equal(o.isinf(), want.isinf())
        fine = want.isfinite()
        assert ((o - want).abs()[fine] <= tol.nan_to_num(0.0)[fine]).all()


@pytest.mark.parametrize("hd,Hkv", [(128, 1), (64, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_a_tile_whose_rows_lie_far_apart(dtype, hd, Hkv):
    """A tile from the first keys to the last of a long context: infinities and NaN of one key or of many, in single
    columns, beside a request that shares the CTAs. (One more look at every key a row and column took seconds.)"""
    n = 100_000
    spread = [0] + list(range(1500, n, 1600)) + [n - 1]
    args = batch([n, 300], [spread, list(range(100, 300))], 4 * Hkv, Hkv, hd, dtype, 64, seed=44)
    q, kc, vc, table, kv, cu, pos = args
    q.mul_(0.25)  # every weight above the smallest f16

    def put(p, col, x, head=0):
        vc[table[0, p // 64].item(), p % 64, head, col] = x

    inf, nan = float("inf"), float("nan")
    for p, col, x in ((70, 0, inf), (40_000, 1, -inf), (40_001, 1, inf), (99_000, hd - 1, nan), (1500, 9, nan),
                      (1501, 10, inf), (63, 17, -inf), (64, 18, -inf), (n - 1, 2, inf)):
        put(p, col, x)
    vc[table[0, 700:760].long(), :, 0, 33] = inf  # 3,840 keys of one column, and all of another key
    vc[table[0, 1200].item(), 5, Hkv - 1] = nan
    want, tol = ref.attend_ref(*args, hd ** -0.5)
    for _ in range(2):
        o = attend(*args, max_q=200).double()
        assert torch.equal(o.isnan(), want.isnan())
        assert torch.equal(o[o.isinf()], want[o.isinf()]) and torch.equal(o.isinf(), want.isinf())
        fine = want.isfinite()
        assert ((o - want).abs()[fine] <= tol.nan_to_num(0.0)[fine]).all()
    assert ops.device_errors() == 0


def test_large_scores():
    """Rows whose maximum grows by far from block to block, and ties at the top."""
    lens = [600, 600]
    args = batch(lens, [[599], list(range(400, 600))], 8, 2, 64, torch.float16, 32, seed=6)
    q, kc = args[0], args[1]
    kc.mul_(8.0)
    q.mul_(4.0)
    check(args, max_qs=(0, 200))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [1, 2 ** 7, 2 ** 15])
def test_scores_of_any_size(dtype, sign, size):
    """Scores of up to 2^30 that float32 holds exactly. The bound is the general one (paged_ref.attend_ref)
    without the scores' rounding, an exponent of d having an error of d e, and 2^-15 for a maximum's rounding
    (log2 units, up to 512) that P may keep."""
    lens = [3000, 700, 300]
    q, kc, vc, table, kv, cu, pos = batch(lens, [[2999], list(range(500, 700)), [100, 299]], 8, 2, 64, dtype, 16, seed=43)
    q.zero_(), kc.zero_()
    q[..., 0] = sign * size
    u, e, rows = torch.finfo(dtype).eps / 2, 2.0 ** -23, []
    for r, n in enumerate(lens):
        m = torch.arange(n, device=DEV)
        slots = table[r, m // 16].long() * 16 + m % 16
        key = (16 * ((m * 7919 + 11) % (n // 2) + 1)).to(dtype)  # two keys of each value (more in bf16), all over
        kc.view(-1, 2, 64)[slots, :, 0] = key[:, None]
        s = sign * size * key.double()
        v = vc.view(-1, 2, 64)[slots].double()
        for i in range(cu[r], cu[r + 1]):
            seen = int(pos[i]) + 1
            d = (s[:seen].max() - s[:seen]) / math.log(2)
            w = torch.softmax(s[:seen], 0)
            out = torch.einsum("m,mgd->gd", w, v[:seen])
            err = w * (u + 2.0 ** -15 + (8 + d) * e + 2 * (seen + 32) * e) + (2.0 ** -25 if dtype == torch.float16 else 0)
            rows.append((out, torch.einsum("m,mgd->gd", err, v[:seen].abs()) + u * out.abs()))
    want, tol = (torch.stack(x).repeat_interleave(4, dim=1) for x in zip(*rows))
    for max_q in (0, 1, 200):
        o = attend(q, kc, vc, table, kv, cu, pos, scale=1.0, max_q=max_q).double()
        assert ((o - want).abs() <= tol).all(), (max_q, (o - want).abs().max().item())
    assert ops.device_errors() == 0


def test_positions_behind_the_last_token_are_flagged_and_see_all():
    args = batch([50], [[49, 50, 1000]], 4, 2, 64, torch.bfloat16, 16, seed=7)
    check(args, max_qs=(0, 3))
    assert ops.device_errors() == N.DEVERR_POSITION


@pytest.mark.parametrize("H", [4, 16])  # 120 and 480 query rows a K/V head: either kernel
def test_missing_pages_are_left_out_and_flagged(H):
    lens = [160, 64]
    for many in (False, True):
        positions = [list(range(100, 160)), [63] * (50 if many else 1)]
        args = batch(lens, positions, H, 2, 64, torch.bfloat16, 16, seed=8)
        q, kc, vc, table, kv, cu, pos = args
        table[0, 3], table[0, 5] = -1, kc.shape[0]
        table[1] = 1 << 20
        o = attend(*args, max_q=60)
        assert ops.device_errors() == N.DEVERR_PAGE
        assert not o[60:].any()
        # the same with the two pages' keys taken out of the row
        keep = [p for p in range(160) if p // 16 not in (3, 5)]
        k = torch.cat([kc[table[0, p // 16].item(), p % 16][None] for p in keep])
        v = torch.cat([vc[table[0, p // 16].item(), p % 16][None] for p in keep])
        n = len(keep)
        k2, v2 = (torch.zeros((-(-n // 16) * 16, 2, 64), dtype=k.dtype, device=DEV) for _ in range(2))
        k2[:n], v2[:n] = k, v
        want, tol = ref.attend_ref(q[:60], k2.view(-1, 16, 2, 64), v2.view(-1, 16, 2, 64),
                                   torch.arange(len(k2) // 16, device=DEV)[None], [n], [0, 60], pos[:60] - 32, 0.125)
        assert ((o[:60].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("H,Hkv,hd", [(16, 4, 128), (8, 8, 64), (6, 2, 96)])
def test_short_runs(H, Hkv, hd, big):
    """Requests of one to eight 16-row tiles, alone and beside one that is larger (they go to different kernels)."""
    lens = [700, 33, 128, 129, 300, 64, 1000]
    count = [5, 8, 16, 1, 31, 2, 40] if G(H, Hkv) > 1 else [17, 33, 100, 1, 16, 2, 128]
    positions = [list(range(max(0, n - c), n)) for n, c in zip(lens, count)]
    if big:
        lens.append(350)
        positions.append(list(range(0, 350)))
    check(batch(lens, positions, H, Hkv, hd, torch.bfloat16, 16, seed=21 + hd), max_qs=(0,))
    assert ops.device_errors() == 0


def G(H, Hkv):
    return H // Hkv


@pytest.mark.parametrize("R,n", [(33, 40), (100, 37), (300, 33)])
def test_many_chunks(R, n):
    """More requests than a warp has lanes, each of several tiles; some without queries, some with one."""
    lens = [n + 7 * (r % 11) for r in range(R)]
    positions = [[] if r % 9 == 4 else [m - 1] if r % 9 == 5 else list(range(m - n, m)) for r, m in enumerate(lens)]
    check(batch(lens, positions, 16, 2, 64, torch.float16, 32, seed=R), max_qs=(n,))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(seed):
    """Runs cut anywhere: random lengths, query counts and order, heads, pages and types."""
    import random
    rng = random.Random(seed)
    H, Hkv, hd = rng.choice(HEADS)
    lens = [rng.randint(1, rng.choice((50, 500, 3000))) for _ in range(rng.randint(1, 12))]
    positions = []
    for m in lens:
        count = rng.choice((0, 1, rng.randint(1, min(m, 40)), rng.randint(1, m)))
        positions.append(sorted(rng.sample(range(m), count)))
    check(batch(lens, positions, H, Hkv, hd, rng.choice((torch.bfloat16, torch.float16)), rng.choice((8, 16, 64, 128)),
                seed=seed, joint=seed % 2 == 0, tail=seed % 3, fill=float("nan")), max_qs=(0,))
    assert ops.device_errors() == 0


def test_long_context():
    """One token and one chunk over 70,001 keys."""
    args = batch([70001], [[70000]], 8, 2, 128, torch.float16, 64, seed=15)
    check(args, max_qs=(1,))
    args = batch([70001], [list(range(69901, 70001))], 8, 2, 64, torch.bfloat16, 64, seed=16)
    check(args, max_qs=(100,))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("width", [1000, 30000, 524287])  # work lists in units of one and of several blocks
def test_wide_tables(width):
    lens = [1, 70, 5000, 9000, 0, 300, 4097, 20000, 64, 640, 33, 1000]
    positions = [[0], [69], [4999], range(8700, 9000), [], range(40), [5, 4096], range(19960, 20000, 3), [63],
                 range(64, 640, 2), [32], [999]]
    args = batch(lens, [list(p) for p in positions], 16, 4, 128, torch.bfloat16, 4096, seed=19)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    table[:, :args[3].shape[1]] = args[3]
    check((*args[:3], table, *args[4:]), max_qs=(0, 300))
    assert ops.device_errors() == 0


@pytest.mark.parametrize("R", [3, 70])
@pytest.mark.parametrize("H", [2, 32])  # 40 and 640 query rows a request and K/V head
def test_offsets_that_do_not_ascend_are_flagged(R, H):
    args = batch([64] * R, [range(24, 64)] * R, H, 2, 64, torch.bfloat16, 16, seed=18)
    q, kc, vc, table, kv, cu, pos = args
    want = attend(*args)
    assert ops.device_errors() == 0
    for bad in ([1] + cu[1:], cu[:-1] + [len(q) + 1], cu[:2] + [cu[1] - 1] + cu[3:], [-1] + cu[1:],
                cu[:2] + [2 ** 31 - 1] + cu[3:], [len(q) * (i % 2) for i in range(R + 1)]):
        for max_q in (0, 1):
            attend(q, kc, vc, table, kv, bad, pos, max_q=max_q)
            assert ops.device_errors() == N.DEVERR_POSITION, bad
    assert torch.equal(attend(*args), want) and ops.device_errors() == 0


def test_lengths_beyond_the_table_are_cut():
    q, kc, vc, table, kv, cu, pos = batch([64], [[63]], 4, 2, 64, torch.bfloat16, 16, seed=17)
    want = attend(q, kc, vc, table, [64], cu, pos)
    assert torch.equal(attend(q, kc, vc, table, [2 ** 31 - 1], cu, pos), want)
    assert ops.device_errors() == 0
    none = attend(q, kc, vc, table[:, :0], [64], cu, pos)  # no page at all
    assert not none.any() and ops.device_errors() == N.DEVERR_POSITION
    none = attend(q, kc[:0], vc[:0], table, [64], cu, pos)  # an empty cache
    assert not none.any() and ops.device_errors() == N.DEVERR_PAGE


def test_strided_operands():
    args = batch([90, 200], [[88, 89], list(range(150, 200))], 8, 2, 64, torch.bfloat16, 16, seed=9)
    q, kc, vc, table, kv, cu, pos = args
    want = attend(*args)
    wide = torch.zeros((q.shape[0], 3, 8, 64), dtype=q.dtype, device=DEV)
    wide[:, 1] = q
    assert torch.equal(attend(wide[:, 1], *args[1:]), want)
    off = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)  # base not on 16 bytes
    off.copy_(q)
    assert torch.equal(attend(off, *args[1:]), want)
    heads_first = kc.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # [pages, Hkv, page, hd] memory
    assert torch.equal(attend(q, heads_first, vc, *args[3:]), want)
    tab = torch.full((2, 40), 10 ** 6, dtype=torch.int32, device=DEV)
    tab[:, :table.shape[1]] = table
    assert torch.equal(attend(q, kc, vc, tab[:, :table.shape[1]], *args[4:]), want)
    assert torch.equal(attend(q, kc, vc, tab, *args[4:]), want)  # a wider table: entries behind kv_lens are not read
    assert ops.device_errors() == 0


def test_results_do_not_depend_on_the_run():
    lens = [3000, 10, 700]
    args = batch(lens, [[2999], list(range(10)), list(range(300, 700))], 16, 4, 128, torch.bfloat16, 64, seed=10)
    first = attend(*args, max_q=400)
    for _ in range(5):
        assert torch.equal(attend(*args, max_q=400), first)


@pytest.mark.parametrize("H,Hkv,hd", [(12, 4, 64), (6, 2, 96), (12, 4, 128), (10, 2, 64), (7, 1, 64), (96, 1, 64)])
def test_results_do_not_depend_on_the_calls_before(H, Hkv, hd):
    """Head groups that do not fill a tile's 128 rows: its other rows must not hold what a call before left in shared
    memory (they share warps with real rows, whose way through the softmax they decide)."""
    wide = 64 if hd <= 64 else 128
    before = batch([600] * 8, [list(range(600))] * 8, 16, 4, wide, torch.bfloat16, 64, seed=49)
    args = batch([900] * 4, [list(range(300, 900, 3))] * 4, H, Hkv, hd, torch.bfloat16, 64, seed=50)
    check(args, max_qs=(200,))
    outs = []
    for x in (float("nan"), 0.0, float("inf"), 3.0e38, 1.0):
        attend(torch.full_like(before[0], x), *before[1:], max_q=600)
        outs.append(attend(*args, max_q=200))
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_offsets_past_32_bits():
    """Pages far into a cache of more than 2^32 bytes."""
    page, Hkv, hd = 64, 4, 128
    pages = 75_000  # 4.9 GB each
    kc = torch.empty((pages, page, Hkv, hd), dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    far = [pages - 1, 2, pages - 7, 70_000]
    for c in (kc, vc):
        for pg in far:
            c[pg] = torch.randn((page, Hkv, hd), device=DEV).to(torch.bfloat16)
    table = i32([far])
    k = torch.randn((1, Hkv, hd), device=DEV).to(torch.bfloat16)
    slot = torch.tensor([(pages - 7) * page + 9], device=DEV)
    ops.rope_paged_write_(k, k, None, None, slot, slot, kc, vc)
    assert torch.equal(kc[pages - 7, 9], k[0]) and torch.equal(vc[pages - 7, 9], k[0])
    for rows in (1, 60):
        q = torch.randn((rows, 16, hd), device=DEV).to(torch.bfloat16)
        pos = torch.arange(256 - rows, 256, device=DEV)
        check((q, kc, vc, table, [256], [0, rows], pos), max_qs=(rows,))
    assert ops.device_errors() == 0


# ---------------------------------------------------------------------------
# streams, graphs, the operators together
# ---------------------------------------------------------------------------


def test_other_stream():
    args = batch([500, 300], [[499], list(range(100, 300))], 8, 2, 128, torch.bfloat16, 16, seed=11)
    want = attend(*args, max_q=200)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = attend(*args, max_q=200)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_calls_at_once():
    """Calls on two streams, in flight together, each with its own workspace."""
    a = batch([9000, 400], [[8999], list(range(200, 400))], 16, 4, 128, torch.bfloat16, 64, seed=18)
    b = batch([7000, 900], [[6999], list(range(100, 900, 2))], 16, 4, 128, torch.bfloat16, 64, seed=19)
    want = [attend(*x, max_q=400) for x in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(attend(*x, max_q=400))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    assert ops.device_errors() == 0


def test_two_graphs_in_turn():
    """Two captured calls replayed in turn on new inputs."""
    a = batch([600, 80], [[599], list(range(80))], 8, 2, 64, torch.bfloat16, 16, seed=22)
    graphs, outs, queries = [], [], [a[0].clone(), a[0].clone()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        attend(*a, max_q=80)
    torch.cuda.synchronize()
    kv, cu = i32(a[4]), i32(a[5])
    pool = torch.cuda.graph_pool_handle()
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(ops.sqdk_paged_fwd(q, a[1], a[2], a[3], kv, cu, a[6], 0.125, 80))
        graphs.append(graph)
    for i in range(6):
        queries[i % 2].copy_(torch.randn(a[0].shape, generator=torch.Generator().manual_seed(i)))
        graphs[i % 2].replay()
        want = attend(queries[i % 2], *a[1:], scale=0.125, max_q=80)
        assert torch.equal(outs[i % 2], want)


def test_captured_step_replays_with_new_lengths():
    """A padded decode step captured once and replayed while requests grow and change."""
    R, P, page, H, Hkv, hd, cap = 4, 12, 16, 8, 2, 64, 6
    g = torch.Generator().manual_seed(12)
    kc, vc = (torch.zeros((60, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.full((R, P), -1, dtype=torch.int32, device=DEV)
    seq, new = i32([0] * R), i32([0] * R)
    free = i32(list(range(60)))
    cos, sin = tables(P * page, hd, torch.float32, g)
    k, v = (torch.zeros((cap, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros((cap, H, hd), dtype=torch.bfloat16, device=DEV)

    def step():
        cu, kv_lens, pos, slots, taken = ops.paged_slots_(table, seq, new, free, page, cap)
        ops.rope_paged_write_(k, v, cos, sin, pos, slots, kc, vc)
        return cu, kv_lens, pos, taken, ops.sqdk_paged_fwd(q, kc, vc, table, kv_lens, cu, pos, 0.125, 3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    held = [0] * R
    for i, lens in enumerate([[1, 3, 0, 2], [1, 0, 1, 1], [2, 1, 1, 1], [0, 0, 1, 0]] * 6):
        seq.copy_(i32(held))
        new.copy_(i32(lens))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        cu, kv_lens, pos, taken, o = out
        held = [a + b for a, b in zip(held, lens)]
        assert kv_lens.tolist() == held
        want, tol = ref.attend_ref(q, kc, vc, table, held, cu.tolist(), pos, 0.125)
        assert ((o.double() - want).abs() <= tol).all() and not o[cu[-1].item():].any()
        free.copy_(torch.roll(free, -taken.item()))
    assert ops.device_errors() == 0


def test_captured_padded_step_with_rotated_queries():
    """A whole step as a user has it, rotation of the queries included, of fewer tokens than it has room for: right,
    and nothing is flagged (the places behind the last token have no position, which rope_gather_rows would flag)."""
    R, P, page, H, Hkv, hd, cap, L = 3, 10, 16, 8, 2, 64, 40, 160
    g = torch.Generator().manual_seed(48)
    kc, vc = (torch.zeros((40, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.full((R, P), -1, dtype=torch.int32, device=DEV)
    seq, new, free = i32([0] * R), i32([0] * R), i32(list(range(40)))
    cos, sin = tables(L, hd, torch.bfloat16, g)
    k, v = (torch.zeros((cap, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros((cap, H, hd), dtype=torch.bfloat16, device=DEV)

    def step():
        cu, kv_lens, pos, slots, taken = ops.paged_slots_(table, seq, new, free, page, cap)
        ops.rope_paged_write_(k, v, cos, sin, pos, slots, kc, vc)
        turned = ops.rope_gather_rows(q[None], pos.clamp(min=0)[None], cos, sin, False)[0]
        return cu, pos, taken, turned, ops.sqdk_paged_fwd(turned, kc, vc, table, kv_lens, cu, pos, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    held, whole = [0] * R, [[] for _ in range(R)]  # each request's keys as they came, not rotated
    u = torch.finfo(torch.bfloat16).eps / 2
    for lens in ([30, 0, 7], [1, 33, 1], [1, 1, 1], [0, 1, 20], [0, 0, 0], [1, 1, 1]):
        seq.copy_(i32(held))
        new.copy_(i32(lens))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        assert ops.device_errors() == 0
        cu, pos, taken, turned, o = out
        n, at = cu[-1].item(), cu.tolist()
        # three roundings of the reference's operations: two products and their sum
        want, size = ref.rope_ref(q[:n], cos, sin, pos[:n])
        assert ((turned[:n].double() - want).abs() <= u * (size + want.abs()) * (1 + 2 * u) + 2.0 ** -120).all()
        held = [a + b for a, b in zip(held, lens)]
        for r in range(R):
            whole[r].append(k[at[r]:at[r + 1]].clone())
            x = torch.cat(whole[r])
            m = torch.arange(held[r], device=DEV)
            got = kc[table[r, m // page].long(), m % page].double()
            want, size = ref.rope_ref(x, cos, sin, m)
            assert ((got - want).abs() <= u * want.abs() * (1 + 1e-6) + 3 * 2.0 ** -24 * size + 2.0 ** -120).all()
        want, tol = ref.attend_ref(turned, kc, vc, table, held, at, pos, 0.125)
        assert ((o.double() - want).abs() <= tol).all() and not o[n:].any()
        free.copy_(torch.roll(free, -taken.item()))
    assert ops.device_errors() == 0


def serve(steps, sync):
    """Steps of slots, write and attention (chunks and single tokens) whose operands the steps before wrote,
    with small kernels and copies of other kinds between them; all that came out."""
    R, H, Hkv, hd, page, pages = 6, 8, 2, 64, 16, 400
    g = torch.Generator().manual_seed(41)
    table = torch.full((R, 70), -1, dtype=torch.int32, device=DEV)
    seq, free = torch.zeros(R, dtype=torch.int32, device=DEV), torch.arange(pages, dtype=torch.int32, device=DEV)
    kc, vc = torch.zeros((2, pages, page, Hkv, hd), dtype=torch.bfloat16, device=DEV)
    x = torch.randn((400, H, hd), generator=g).to(torch.bfloat16).to(DEV)
    new = [torch.randint(0, 1 + most, (R,), generator=g, dtype=torch.int32).to(DEV) for most in (60, 1, 5, 1) * steps]
    wait = torch.cuda.synchronize if sync else lambda: None
    out = []
    for lens in new:
        wait()
        cu, kv, pos, slots, taken = ops.paged_slots_(table, seq, lens, free, page, 400)
        wait()
        ops.rope_paged_write_(x[:, :Hkv], x[:, Hkv:2 * Hkv], None, None, pos, slots, kc, vc)
        wait()
        o = ops.sqdk_paged_fwd(x, kc, vc, table, kv, cu, pos, 0.125)
        wait()
        out.append(o)
        x = torch.where(pos[:, None, None] >= 0, o + x, x) * 0.7
        seq.copy_(kv)
        free = free.gather(0, (torch.arange(pages, device=DEV) + taken) % pages)  # no page is given twice
    return out, kc, vc, table


def test_steps_in_a_row_equal_steps_one_by_one():
    one_by_one = serve(12, True)
    for _ in range(4):
        in_a_row = serve(12, False)
        assert all(torch.equal(a, b) for a, b in zip(one_by_one[0], in_a_row[0]))
        assert all(torch.equal(a, b) for a, b in zip(one_by_one[1:], in_a_row[1:]))


def test_capture_between_other_nodes():
    """Operators captured behind a memset, a copy and a joined stream."""
    lens = [33, 200]
    q, kc, vc, table, kv, cu, pos = batch(lens, [[32], list(range(100, 200))], 8, 2, 64, torch.bfloat16, 16, seed=42)
    kv_, cu_ = i32(kv), i32(cu)
    want = ops.sqdk_paged_fwd(q, kc, vc, table, kv_, cu_, pos, 0.125)
    q2, kv2, stamp, k2 = torch.empty_like(q), torch.empty_like(kv_), torch.ones(8, device=DEV), torch.zeros_like(kc)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        stamp.zero_()
        q2.copy_(q)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            kv2.copy_(kv_)
            k2.copy_(kc)
        first = ops.sqdk_paged_fwd(q, kc, vc, table, kv_, cu_, pos, 0.125)
        main.wait_stream(side)
        second = ops.sqdk_paged_fwd(q2, k2, vc, table, kv2, cu_, pos, 0.125)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            third = ops.sqdk_paged_fwd(q2, k2, vc, table, kv2, cu_, pos, 0.125, 1)
        main.wait_stream(side)
    one = torch.empty_like(third)
    for _ in range(3):
        for t in (q2, kv2, k2, first, second, third):
            t.zero_()
        g.replay()
        one.copy_(third)
        assert torch.equal(first, want) and torch.equal(second, want)
        assert not stamp.any() and ((one.double() - want.double()).abs() <= 2.0 ** -6 * want.double().abs() + 2.0 ** -8).all()


def test_prefill_in_chunks_and_decode_equal_the_whole_sequence():
    """Prompts brought in chunk by chunk and then token by token give what sqdk_fwd gives on the whole sequence."""
    B, S, H, Hkv, hd, page = 3, 200, 8, 2, 64, 16
    g = torch.Generator().manual_seed(13)
    q, k, v = (torch.randn((B, S, h, hd), generator=g).to(torch.bfloat16).to(DEV) for h in (H, Hkv, Hkv))
    cos, sin = tables(S, hd, torch.float32, g)
    kc, vc = (torch.full((64, page, Hkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.full((B, -(-S // page)), -1, dtype=torch.int32, device=DEV)
    free = i32(torch.randperm(64, generator=g).tolist())
    held, rows = [0] * B, [[] for _ in range(B)]
    plan = [[70, 1, 33], [0, 100, 64], [60, 64, 1]] + [[1, 1, 1]] * 35
    for new in plan:
        pick = [slice(h, h + m) for h, m in zip(held, new)]
        cu, kv_lens, pos, slots, taken = ops.paged_slots_(table, i32(held), i32(new), free, page, sum(new))
        ops.rope_paged_write_(torch.cat([k[b, s] for b, s in enumerate(pick)]),
                              torch.cat([v[b, s] for b, s in enumerate(pick)]), cos, sin, pos, slots, kc, vc)
        o = ops.sqdk_paged_fwd(torch.cat([q[b, s] for b, s in enumerate(pick)]), kc, vc, table, kv_lens, cu, pos, 0.125,
                               max(new))
        free = free[taken.item():]
        at = 0
        for b, m in enumerate(new):
            rows[b].append(o[at:at + m])
            at += m
        held = [h + m for h, m in zip(held, new)]
    n = min(held)
    assert n == 133
    got = torch.stack([torch.cat(r)[:n] for r in rows])
    rot = torch.stack([ref.rope_ref(k[b, :n], cos, sin, torch.arange(n, device=DEV))[0] for b in range(B)]).to(torch.bfloat16)
    idx = torch.arange(n, device=DEV).expand(B, n).contiguous()
    dense = ops.sqdk_fwd(q[:, :n].contiguous(), rot, v[:, :n].contiguous(), idx, 0.125)
    want, tol = ref.attend_ref(q[:, :n].reshape(-1, H, hd), rot.view(B, n, Hkv, hd), v[:, :n],
                               torch.arange(B, device=DEV)[:, None], [n] * B, [0, n, 2 * n, 3 * n], idx.reshape(-1), 0.125)
    assert ((got.reshape(-1, H, hd).double() - want).abs() <= tol).all()
    # two kernels, each within its bound
    assert ((got - dense).double().abs().reshape(-1, H, hd) <= 2 * tol + 2.0 ** -8 * want.abs()).all()
    assert ops.device_errors() == 0


def test_writes_raise_the_version_of_what_they_write():
    n, Hkv, hd, page = 3, 2, 64, 16
    kv = torch.zeros((4, 2, page, Hkv, hd), dtype=torch.bfloat16, device=DEV)
    kc, vc = kv[:, 0], kv[:, 1]
    k = torch.randn((n, Hkv, hd), device=DEV).to(torch.bfloat16)
    slots = torch.arange(n, device=DEV)
    lens = i32([0])
    for write, make in ((ops.rope_paged_write_, ops.paged_slots_),
                        (torch.ops.hspmn.rope_paged_write_, torch.ops.hspmn.paged_slots_)):
        apart = [torch.zeros_like(kc) for _ in range(2)]
        table = i32([[-1, -1]])
        before = [t._version for t in (kv, *apart, table, k, slots, lens)]
        write(k, k, None, None, slots, slots, kc, vc)
        write(k, k, None, None, slots, slots, *apart)
        make(table, lens, i32([3]), i32([0]), page, n)
        after = [t._version for t in (kv, *apart, table, k, slots, lens)]
        assert all(b > a for a, b in zip(before[:4], after[:4])) and before[4:] == after[4:]
    assert ops.device_errors() == 0


def test_backward_over_an_overwritten_cache_raises():
    page, Hkv, hd = 16, 2, 64
    kc, vc = (torch.randn((2, page, Hkv, hd), device=DEV).to(torch.bfloat16) for _ in range(2))
    k = torch.randn((3, Hkv, hd), device=DEV).to(torch.bfloat16)
    slots = torch.arange(3, device=DEV)
    q = torch.randn((2, 5, 4, hd), device=DEV).to(torch.bfloat16).requires_grad_()
    idx = torch.arange(5, device=DEV).expand(2, 5).contiguous()
    for graph in (lambda: (q[:, :1, :Hkv] * kc).sum(), lambda: ops.sqdk_attention(q, kc, vc, idx, 0.125).float().sum()):
        graph().backward()  # nothing written in between
        y = graph()
        ops.rope_paged_write_(k, k, None, None, slots, slots, kc, vc)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    table = i32([[-1, 5]])
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = w[table.clamp(min=0).long()].sum() + (w[:2] * table).sum()
    ops.paged_slots_(table, i32([0]), i32([3]), i32([0]), page, 3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_derivatives_that_would_be_dropped_are_refused():
    """Learned tables, and forward-mode tangents of any operand: there is no derivative, so none is dropped in silence."""
    import torch.autograd.forward_ad as fw
    page, Hkv, hd = 16, 2, 64
    kc, vc = (torch.zeros((2, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    x = torch.randn((3, Hkv, hd), device=DEV).to(torch.bfloat16)
    cos = torch.ones((8, hd), dtype=torch.float32, device=DEV)
    at = torch.arange(3, device=DEV)
    table, kv, cu = i32([[0, 1]]), i32([3]), i32([0, 3])
    for cos_, sin_ in ((cos.clone().requires_grad_(), cos), (cos, cos.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no backward"):
            ops.rope_paged_write_(x, x, cos_, sin_, at, at, kc, vc)
        with torch.no_grad():
            ops.rope_paged_write_(x, x, cos_, sin_, at, at, kc, vc)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))

        args = (x, x, cos, cos, at, at, kc, vc)
        for i in (0, 1, 2, 3, 6, 7):
            for grad_mode in (torch.enable_grad, torch.no_grad):
                with grad_mode(), pytest.raises(RuntimeError, match="forward-mode"):
                    ops.rope_paged_write_(*args[:i], dual(args[i]), *args[i + 1:])
        args = (x, kc, vc, table, kv, cu, at, 0.125)
        for i in range(3):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.sqdk_paged_fwd(*args[:i], dual(args[i]), *args[i + 1:])
        ops.sqdk_paged_fwd(*args)
        with fw._set_fwd_grad_enabled(False):
            ops.sqdk_paged_fwd(dual(x), *args[1:])
    assert ops.device_errors() == 0


def test_caches_made_in_inference_mode():
    n, Hkv, hd, page = 3, 2, 64, 16
    k = torch.randn((n, Hkv, hd), device=DEV).to(torch.bfloat16)
    slots, free = torch.arange(n, device=DEV), i32([0])
    with torch.inference_mode():
        kc, vc = (torch.zeros((1, page, Hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        table = i32([[-1]])
        ops.rope_paged_write_(k, k, None, None, slots, slots, kc, vc)
        ops.paged_slots_(table, i32([0]), i32([n]), free, page, n)
    assert torch.equal(kc[0, :n], k) and table.tolist() == [[0]]
    ops.rope_paged_write_(-k, k, None, None, slots, slots, kc, vc)  # and outside, as before
    ops.paged_slots_(table, i32([0]), i32([n]), free, page, n)
    assert torch.equal(kc[0, :n], -k)


def test_refusals():
    q, kc, vc, table, kv, cu, pos = batch([20], [[18, 19]], 4, 2, 64, torch.bfloat16, 16, seed=23)
    kv, cu = i32(kv), i32(cu)

    def fwd(q=q, kc=kc, vc=vc, table=table, kv=kv, cu=cu, pos=pos, scale=0.125, max_q=0):
        return ops.sqdk_paged_fwd(q, kc, vc, table, kv, cu, pos, scale, max_q)

    fwd()
    for over in (dict(q=q[0]), dict(kc=kc[0]), dict(kc=kc[:, :8]), dict(kc=kc[..., :32], vc=vc[..., :32]),
                 dict(table=table[0]), dict(table=table.long()), dict(kv=kv.long()), dict(kv=kv[:0]), dict(cu=cu[:1]),
                 dict(pos=pos[:1]), dict(pos=pos.int()), dict(q=q[:, :3]),
                 dict(kc=kc.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            fwd(**over)
    for over in (dict(q=q.float()), dict(q=q.half()), dict(vc=vc.half())):
        with pytest.raises(TypeError):
            fwd(**over)
    for over in (dict(scale=-1.0), dict(scale=float("inf")), dict(max_q=-1), dict(kc=kc[:, :12], vc=vc[:, :12])):
        with pytest.raises(N.HSPMNNativeError):
            fwd(**over)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fwd(pos=pos.cpu())
    with pytest.raises(RuntimeError, match="no backward"):
        fwd(q=q.clone().requires_grad_())
    with torch.no_grad():
        fwd(q=q.clone().requires_grad_())

    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=DEV)
    cos = torch.zeros((32, 64), dtype=torch.bfloat16, device=DEV)

    def write(k=k, v=k, cos=cos, sin=cos, pos=pos, slots=pos, kc=kc, vc=vc):
        ops.rope_paged_write_(k, v, cos, sin, pos, slots, kc, vc)

    write()
    write(k=k[:0], v=k[:0], pos=pos[:0], slots=pos[:0])
    for over in (dict(k=k[0], v=k[0]), dict(v=k[:1]), dict(sin=None), dict(cos=cos[:, :32], sin=cos[:, :32]), dict(sin=cos[:5]),
                 dict(pos=pos[:1]), dict(slots=pos.int()), dict(kc=kc[:, :, :1], vc=vc[:, :, :1])):
        with pytest.raises(ValueError):
            write(**over)
    for over in (dict(v=k.half()), dict(cos=cos.half(), sin=cos.half()), dict(kc=kc.half()), dict(k=k.double(), v=k.double())):
        with pytest.raises(TypeError):
            write(**over)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        write(cos=cos.cpu(), sin=cos.cpu())
    with pytest.raises(RuntimeError, match="no backward"):
        write(k=k.clone().requires_grad_())

    t = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    n = i32([1, 2])
    ops.paged_slots_(t, n, n, n, 16, 3)
    for args in ((t[0], n, n, n, 16, 3), (t, n[:1], n, n, 16, 3), (t, n, n.long(), n, 16, 3), (t, n, n, t, 16, 3),
                 (t, n, n, n, 16, -1), (t.t().contiguous().t(), n, n, n, 16, 3), (t[:1].expand(2, 4), n, n, n, 16, 3)):
        with pytest.raises(ValueError):
            ops.paged_slots_(*args)
    with pytest.raises(N.HSPMNNativeError):
        ops.paged_slots_(t, n, n, n, 20, 3)
    assert ops.device_errors() == 0


def test_calls_are_counted_and_timed():
    q, kc, vc, table, kv, cu, pos = batch([20], [[19]], 4, 2, 64, torch.bfloat16, 16, seed=24)
    before = ops.LaunchStats.launches
    with ops.KernelTimer() as timer:
        attend(q, kc, vc, table, kv, cu, pos)
    torch.cuda.synchronize()
    assert timer.results()["sqdk_paged_fwd"]["launches"] == 1 and ops.LaunchStats.launches == before + 1
    attend(q, kc, vc, table, kv, cu, pos)
    assert ops.LaunchStats.launches == before + 2


def test_compiled_step_is_one_graph():
    q, kc, vc, table, kv, cu, pos = batch([20, 50], [[19], [49]], 4, 2, 64, torch.bfloat16, 16, seed=25)
    kv, cu = i32(kv), i32(cu)

    def step(q, kc, vc):
        return ops.sqdk_paged_fwd(q * 2, kc, vc, table, kv, cu, pos, 0.125, 1) + 1

    got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, kc, vc)
    assert torch.equal(got, step(q, kc, vc))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_serving_step(backend):
    """The three operators in one graph: tables and caches that are its inputs are written in place, as eager calls
    write them, and so are tensors that it makes itself."""
    R, page, Hkv, H, hd, n = 2, 16, 2, 8, 64, 25
    g = torch.Generator().manual_seed(46)
    k, v = (torch.randn((n, Hkv, hd), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn((n, H, hd), generator=g).to(torch.bfloat16).to(DEV)
    cos, sin = tables(64, hd, torch.float32, g)
    free = i32([3, 1, 5, 0])
    caches = torch.randn((2, 6, page, Hkv, hd), generator=g).to(torch.bfloat16).to(DEV)

    def step(table, kc, vc, seq, new, k, v, q):
        cu, kv, pos, slots, taken = ops.paged_slots_(table, seq, new, free, page, n)
        ops.rope_paged_write_(k * 2, v, cos, sin, pos, slots, kc, vc)
        own_k, own_v = kc + 1, torch.zeros_like(vc)
        ops.rope_paged_write_(k, v, None, None, pos, slots, own_k, own_v)
        return (ops.sqdk_paged_fwd(q + 1, kc, vc, table, kv, cu, pos, 0.125, 20), own_k.sum(), own_v, cu, kv, pos, slots,
                taken)

    def run(f):
        table, (kc, vc) = i32([[4, -1, -1], [-1, -1, 9]]), caches.clone()
        out = f(table, kc, vc, i32([9, 0]), i32([20, 4]), k, v, q)
        return (*out, table, kc, vc)

    want = run(step)
    compiled = torch.compile(step, backend=backend, fullgraph=True)
    for _ in range(2):
        for a, b in zip(run(compiled), want):
            assert torch.equal(a, b)
    assert want[-3].tolist() == [[4, 3, -1], [1, -1, 9]]
    assert ops.device_errors() == 0


def test_compiled_step_takes_any_max_q():
    from torch._dynamo.testing import CompileCounterWithBackend
    args = batch([20, 50], [[19], [49, 48, 47]], 4, 2, 64, torch.bfloat16, 16, seed=47)
    q, kc, vc, table, kv, cu, pos = args
    kv, cu = i32(kv), i32(cu)
    counter = CompileCounterWithBackend("aot_eager")
    step = torch.compile(lambda m: ops.sqdk_paged_fwd(q, kc, vc, table, kv, cu, pos, 0.125, m), backend=counter, fullgraph=True)
    for m in (3, 4, 5, 9, 60):
        assert torch.equal(step(m), ops.sqdk_paged_fwd(q, kc, vc, table, kv, cu, pos, 0.125, m))
    assert counter.frame_count <= 2  # the first value, and any other


def test_registered_operators_trace():
    args = batch([20], [[19]], 4, 2, 64, torch.bfloat16, 16, seed=14)
    q, kc, vc, table, kv, cu, pos = args
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.hspmn.sqdk_paged_fwd.default, (q, kc, vc, table, i32(kv), i32(cu), pos, 0.125, 1),
                          test_utils=checks)
    torch.library.opcheck(torch.ops.hspmn.paged_slots_.default, (table, i32([16]), i32([4]), i32([0, 1]), 16, 4),
                          test_utils=checks)
    k = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=DEV)
    torch.library.opcheck(torch.ops.hspmn.rope_paged_write_.default, (k, k, None, None, pos, pos, kc, vc),
                          test_utils=checks)
