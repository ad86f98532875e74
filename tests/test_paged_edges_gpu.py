"""Edges of the paged 4-bit cache's operators on the GPU: lengths and page ids that no server sends, queries, keys and values
of very different sizes, pages freed behind a window, batches that break their bounds -- each in every form of the attention
that a call can take (tests/paged_reference.py holds the plain statements in 64 bits)."""

import math

import pytest

from tests import paged_reference as R
from tests.test_paged_gpu import BOUNDS, _attend, _cache, _gen, _i32, _status

pytestmark = pytest.mark.gpu


# ---- plan ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cached,new", [
    ([2 ** 31 - 1, 9], [1, 3]),                    # the page count of the first would wrap around
    ([2 ** 31 - 1, 9], [2 ** 31 - 1, 3]),
    ([2 ** 30, 9], [2 ** 31 - 1, 3]),
    ([0, 9], [2 ** 31 - 1, 3]),
    ([2 ** 31 - 65537, 2 ** 31 - 65537, 9], [5, 2 ** 31 - 1, 3]),
    ([-2 ** 31, 5, 9], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]),
])
@pytest.mark.parametrize("page", [8, 65536])
def test_plan_lengths_beyond_31_bits(cuda, cached, new, page):
    """Nothing is written outside the requests' table rows, positions never wrap around, and sums stop at 2^31 - 1."""
    import torch
    from locals_b200 import paged

    B, width, tokens, most = len(cached), 4, 9, 2 ** 31 - 1
    whole = torch.full((B + 64, width), -7, dtype=torch.int32, device=cuda)
    table = whole[32:32 + B]
    free = torch.arange(100, 200, dtype=torch.int32, device=cuda)
    p = paged.plan(_i32(cached, cuda), _i32(new, cuda), table, free, _i32([1], cuda), page, tokens)
    assert _status() == BOUNDS
    assert bool((whole[:32] == -7).all()) and bool((whole[32 + B:] == -7).all())
    far, lens, start, pages = most - 65536, [], [0], 0
    for c, n in zip(cached, new):
        c = min(max(c, 0), far)
        n = min(max(n, 0), far - c)
        lens.append(c + n)
        start.append(min(start[-1] + n, most))
        pages = min(pages + -(-(c + n) // page) - -(-c // page), most)
    assert p.lens.tolist() == lens and p.q_start.tolist() == start and p.head.item() == min(1 + pages, most)
    for t, (pos, slot) in enumerate(zip(p.positions.tolist(), p.slots.tolist())):
        if t >= start[-1]:
            assert (pos, slot) == (0, -1)
            continue
        b = max(i for i in range(B) if start[i] <= t)
        assert pos == min(max(cached[b], 0), far) + t - start[b]
        if slot >= 0:
            col = pos // page
            assert col < width and slot % page == pos % page
            assert slot // page == table[b, col].item()


def test_plan_page_ids_beyond_any_pool(cuda):
    """An id whose slots are beyond 31 bits gets none of them: not a slot that its product wraps around to."""
    import torch
    from locals_b200 import paged

    table = _i32([[2 ** 26 + 3, 5], [2 ** 31 - 1, -1]], cuda)
    free = _i32([2 ** 27 + 1, 2 ** 27 - 1], cuda)
    p = paged.plan(_i32([62, 0], cuda), _i32([4, 0], cuda), table, free, _i32([0], cuda), 64, 4)
    # request 0: places 62 and 63 of an id beyond, then the second column is its own new page free[0], beyond too
    assert p.positions.tolist() == [62, 63, 64, 65] and p.slots.tolist() == [-1, -1, -1, -1]
    assert _status() == BOUNDS
    last = 2 ** 31 // 16 - 1  # the last id whose slots fit
    p = paged.plan(_i32([0], cuda), _i32([16], cuda), _i32([[-1]], cuda), _i32([last], cuda), _i32([0], cuda), 16, 16)
    assert p.slots.tolist() == list(range(2 ** 31 - 16, 2 ** 31)) and _status() == 0


@pytest.mark.parametrize("B", [6127, 6128, 6143, 6144])
def test_plan_of_any_batch_in_a_new_process(B):
    """A process's first plan, at the sizes around the default limit of shared memory."""
    import subprocess
    import sys

    code = ("import torch\nfrom locals_b200 import paged\n"
            f"B = {B}\ni = lambda *s, v=0: torch.full(s, v, dtype=torch.int32, device='cuda')\n"
            "p = paged.plan(i(B), i(B, v=1), i(B, 1, v=-1), torch.arange(B, dtype=torch.int32, device='cuda'), i(1), 16, B)\n"
            "assert p.slots.tolist() == [16 * b for b in range(B)]\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-500:]


# ---- attend: bounds of a batch -----------------------------------------------------------------------

@pytest.mark.parametrize("columns", [0, 9000])
def test_attend_more_queries_than_max_q(cuda, columns):
    """The first max_q of a request's queries stand where they stand; its others, rows before q_start[0] and rows past
    q_start[-1] are 0."""
    import torch
    from locals_b200 import paged

    g = _gen(cuda, 5)
    lens, H, KVH, D = [300, 90, 41], 8, 2, 128
    keys, values, table = _cache(cuda, lens, KVH, D, 16, "bfloat16", 5)
    table = torch.cat([table, torch.full((3, columns), -1, dtype=torch.int32, device=cuda)], 1)
    start, most = [3, 53, 54, 94], 40  # 50, 1 and 40 queries
    q = torch.randn((100, H, D), generator=g, device=cuda).to(torch.bfloat16)
    torch.full((4, 100, H, D), float("nan"), device=cuda)  # (what the output's memory may hold)
    got = paged.attend(q, keys, values, table, _i32(lens, cuda), 0.1, q_start=_i32(start, cuda), max_q=most)
    assert _status() == BOUNDS
    ref, bound = R.attended(q, keys, values, table, _i32(lens, cuda), 0.1, _i32(start, cuda), None, 0)
    ref[3 + most:53], bound[3 + most:53] = 0, 0
    assert bool(((got.double() - ref).abs() <= bound).all())
    for rows in (got[:3], got[3 + most:53], got[94:]):
        assert torch.count_nonzero(rows).item() == 0


@pytest.mark.parametrize("new,columns,H,D", [(1, 0, 8, 128), (3, 0, 8, 64), (40, 9000, 8, 128), (140, 9000, 8, 128),
                                             (60, 9000, 4, 256), (140, 9000, 4, 256)])
def test_attend_pages_freed_behind_a_window(cuda, new, columns, H, D):
    """Table entries wholly behind the window may be -1, or anything: no key there is missed."""
    import torch
    from locals_b200 import paged

    n, page, window = 1000, 16, 333
    got, (q, keys, values, table, qs, scale, _) = _attend(cuda, [new], [n], H, 2, D, page, "bfloat16", window, seed=9,
                                                          columns=columns, max_q=new)
    freed = table.clone()
    behind = max(0, n - new + 1 - window) // page
    assert behind > 20
    freed[0, :behind] = -1
    again = paged.attend(q, keys, values, freed, _i32([n], cuda), scale, q_start=qs, max_q=new, window=window)
    assert _status() == 0
    assert torch.equal(again, got)


# ---- attend: sizes -----------------------------------------------------------------------------------

FORMS = [  # new, query heads, kv heads, head_dim, columns of 16 keys
    (5, 8, 2, 128, 0),        # few rows, a cluster an item
    (5, 8, 2, 128, 9000),     # few rows, the even split
    (5, 8, 2, 64, 9000),
    (5, 8, 2, 256, 9000),
    (40, 8, 2, 128, 9000),    # many rows, unpacked in place
    (140, 8, 2, 64, 9000),    # many rows, unpacked first
    (140, 8, 2, 128, 9000),
    (40, 8, 2, 256, 9000),
    (140, 8, 2, 256, 9000),
]


def _case(cuda, new, H, KVH, D, columns, seed, n=300, dtype="bfloat16"):
    import torch

    g = _gen(cuda, seed)
    keys, values, table = _cache(cuda, [n], KVH, D, 16, dtype, seed)
    table = torch.cat([table, torch.full((1, columns), -1, dtype=torch.int32, device=cuda)], 1)
    q = (1.5 * torch.randn((new, H, D), generator=g, device=cuda)).to(getattr(torch, dtype))
    return q, keys, values, table, _i32([n], cuda), _i32([0, new], cuda)


def _held(q, keys, values, table, lens, scale, qs, sinks=None, window=0):
    """The attention, checked against the 64-bit statement where that is a number."""
    import torch
    from locals_b200 import paged

    got = paged.attend(q, keys, values, table, lens, scale, q_start=qs, max_q=q.shape[0], sinks=sinks, window=window)
    ref, bound = R.attended(q, keys, values, table, lens, scale, qs, sinks, window)
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), f"beyond the bound by {off.max().item()}, {(got.double() - ref).abs().max().item()} in all"
    return got


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_a_query_of_any_size_moves_no_other_row(cuda, new, H, KVH, D, columns):
    import torch
    from locals_b200 import paged

    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 21)
    got = _held(q, keys, values, table, lens, D ** -0.5, qs)
    for bad in (math.inf, -math.inf, math.nan, 2.0 ** 100, -2.0 ** 40):
        poisoned = q.clone()
        poisoned[new - 1, 2, 7] = bad  # the last token's third head
        again = paged.attend(poisoned, keys, values, table, lens, D ** -0.5, q_start=qs, max_q=new)
        same = torch.ones_like(q, dtype=torch.bool)
        same[new - 1, 2] = False
        assert torch.equal(again[same], got[same]), bad
        if not math.isfinite(bad):
            assert not bool(torch.isfinite(again[new - 1, 2].float()).all())


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_queries_of_very_different_sizes(cuda, new, H, KVH, D, columns):
    """Rows 2^-30 to 2^30 times the usual: each is held to its own size (a large one's largest score takes all)."""
    import torch

    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 22)
    size = 2.0 ** torch.linspace(-30, 0, new * H, device=q.device).round().view(new, H, 1)
    _held((q.float() * size).to(q.dtype), keys, values, table, lens, D ** -0.5, qs)
    # both inverse sizes at once: the scores are ordinary ones again
    for e in (20, -20, 110, -110):
        _held((q.float() * 2.0 ** e).to(q.dtype), keys, values, table, lens, D ** -0.5 * 2.0 ** -e, qs)


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_a_sink_that_is_not_a_number(cuda, new, H, KVH, D, columns):
    """It makes its own head NaN and no other; a query that sees nothing stays 0."""
    import torch
    from locals_b200 import paged

    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 27)
    sinks = torch.linspace(-1, 1, H, device=q.device)
    got = _held(q, keys, values, table, lens, D ** -0.5, qs, sinks)
    sinks[3] = math.nan
    again = paged.attend(q, keys, values, table, lens, D ** -0.5, q_start=qs, max_q=new, sinks=sinks)
    assert bool(torch.isnan(again[:, 3]).all())
    others = [h for h in range(H) if h != 3]
    assert torch.equal(again[:, others], got[:, others])
    none = paged.attend(q, keys, values, table, _i32([0], q.device), D ** -0.5, q_start=qs, max_q=new, sinks=sinks)
    assert torch.count_nonzero(none).item() == 0


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_keys_of_any_size(cuda, new, H, KVH, D, columns):
    """Keys of 2^-60 to 2^20 of the usual size met by queries of the inverse size; and one group of 64 dimensions of the keys
    2^-16 of the others, its queries 2^16 of theirs: all scores as they were."""
    import torch

    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 23)
    for e in (-8, -12, -16, -60, 14, 20):
        small = (keys[0], keys[1] * 2.0 ** e, keys[2] * 2.0 ** e)
        _held(q * 2.0 ** -e, small, values, table, lens, D ** -0.5, qs)
    if D > 64:
        s, b, x = keys[1].clone(), keys[2].clone(), q.clone()
        s[..., 1] *= 2.0 ** -16
        b[..., 1] *= 2.0 ** -16
        x[..., 64:128] *= 2.0 ** 16
        _held(x, (keys[0], s, b), values, table, lens, D ** -0.5, qs)


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_value_groups_of_any_size(cuda, new, H, KVH, D, columns):
    """A group of 64 dimensions of the values 2^-6 to 2^-14 of the others: its outputs are held to their own size."""
    import torch

    if D == 64:
        pytest.skip("one group a head")
    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 24)
    for e, all_e in ((-6, -5), (-10, 0), (-14, 0), (-14, 8)):
        s, b = values[1] * 2.0 ** all_e, values[2] * 2.0 ** all_e
        s[..., 1] *= 2.0 ** e
        b[..., 1] *= 2.0 ** e
        _held(q, keys, (values[0], s, b), table, lens, D ** -0.5, qs)


@pytest.mark.parametrize("new,H,KVH,D,columns", FORMS)
def test_attend_values_that_grow_and_shrink_along_the_keys(cuda, new, H, KVH, D, columns):
    """Keys in runs of 64 whose values are 2^-40 to 2^100 of the usual size, in every order: finite, and within the bound."""
    import torch

    q, keys, values, table, lens, qs = _case(cuda, new, H, KVH, D, columns, 25, n=640)
    for sizes in ([0, 2, -3, 6, 9, -8, 1, 0, -2, 5], [100, 0, -40, 3, 0, 100, -40, 0, 8, 20], [-40, 0, 100, 0, -40, 0, 0, 0, 0, 0],
                  [0, -40, -40, 0, 0, 0, -20, 0, 0, 10], [100, 100, -40, -40, 0, 0, -40, -40, 0, 0]):
        s, b = values[1].clone(), values[2].clone()
        for r, e in enumerate(sizes):
            ids = table[0, 4 * r:4 * r + 4].long()
            s[ids] *= 2.0 ** e
            b[ids] *= 2.0 ** e
        _held(q, keys, (values[0], s, b), table, lens, D ** -0.5, qs)
