"""The forms that attention over the paged 4-bit cache can take -- which one a call's sizes select (lq_kv4_attend_forms), and
edge cases on each by name, so that a change of the rules cannot take a test elsewhere unseen."""

import math

import pytest

from tests import paged_reference as R
from tests.test_paged_gpu import BOUNDS, _attend, _i32, _status

pytestmark = pytest.mark.gpu

CLUSTERS, SPLIT, TILES, DENSE = 1, 2, 4, 8

# form, new tokens, query heads, kv heads, head_dim, table columns (16 keys each) beyond the requests' own
EACH = [
    (CLUSTERS, 5, 8, 2, 128, 0),
    (SPLIT, 5, 8, 2, 64, 9000),
    (SPLIT, 5, 8, 2, 128, 9000),
    (SPLIT, 5, 8, 2, 256, 9000),
    (TILES, 40, 8, 2, 64, 9000),
    (TILES, 40, 8, 2, 128, 9000),
    (TILES, 40, 8, 2, 256, 9000),
    (DENSE, 140, 8, 2, 64, 9000),
    (DENSE, 140, 8, 2, 128, 9000),
    (DENSE, 140, 8, 2, 256, 9000),
]
FORMS = pytest.mark.parametrize("form,new,H,KVH,D,columns", EACH)


def _forms(B, max_q, H, KVH, D, width, page=16, window=0):
    from locals_b200 import _lib

    return _lib.lib().lq_kv4_attend_forms(B, max_q, H, KVH, D, width, page, window)


def _one(cuda, form, new, n, H, KVH, D, columns, dtype="bfloat16", **more):
    got, state = _attend(cuda, [new], [n], H, KVH, D, 16, dtype, columns=columns, max_q=new, **more)
    took = _forms(1, new, H, KVH, D, state[3].shape[1], window=more.get("window", 0))
    assert took & form or (form == SPLIT and more.get("window") and took == CLUSTERS)  # (a window keeps the steps few)
    return got, state


def test_forms_by_sizes(cuda):
    assert _forms(1, 1, 32, 8, 128, 63) == CLUSTERS
    assert _forms(64, 1, 32, 4, 128, 512) == SPLIT
    assert _forms(4, 1, 32, 4, 128, 2048, 64) == SPLIT
    assert _forms(4, 1, 32, 4, 128, 2048, 64, 300) == CLUSTERS  # a window keeps the steps few
    assert _forms(8, 1024, 32, 8, 128, 192) == CLUSTERS | DENSE  # decoding requests beside prompts
    assert _forms(1, 4096, 16, 2, 128, 2048) == SPLIT | DENSE
    assert _forms(1, 4096, 16, 2, 128, 200000) == SPLIT | TILES  # more room than the unpacked tiles may take
    assert _forms(1, 300, 20, 1, 128, 9000) == DENSE             # 20 heads of one query are more than a tile of few rows
    for refused in ((0, 1, 8, 2, 128, 4), (1, 0, 8, 2, 128, 4), (1, 1, 9, 2, 128, 4), (1, 1, 8, 2, 96, 4), (1, 1, 8, 2, 128, 0)):
        assert _forms(*refused) == 0


@FORMS
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_each_form(cuda, form, new, H, KVH, D, columns, dtype):
    for n, window, sinks in ((new, 0, False), (333, 0, True), (700, 129, False), (700, 1, True)):
        _one(cuda, form, new, n, H, KVH, D, columns, dtype, window=window, sinks=sinks, seed=n)


@FORMS
@pytest.mark.parametrize("scale", [40.0, 0.0, -1.0])
def test_scales(cuda, form, new, H, KVH, D, columns, scale):
    _one(cuda, form, new, 300, H, KVH, D, columns, scale=scale, seed=6)


@FORMS
def test_sinks_of_any_size(cuda, form, new, H, KVH, D, columns):
    import torch
    from locals_b200 import paged

    plain, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, 300, H, KVH, D, columns, seed=8)
    for level, same in ((-math.inf, True), (-3e38, True), (3e38, False), (math.inf, False)):
        sinks = torch.full((H,), level, device=cuda)
        got = paged.attend(q, keys, values, table, _i32([300], cuda), scale, q_start=qs, max_q=new, sinks=sinks)
        assert torch.equal(got, plain) if same else torch.count_nonzero(got).item() == 0


@FORMS
def test_masked_places_may_hold_anything(cuda, form, new, H, KVH, D, columns):
    import torch
    from locals_b200 import paged

    got, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, 300, H, KVH, D, columns, seed=9)
    page, off = int(table[0, 299 // 16]), 299 % 16
    for bad in (math.nan, math.inf, -math.inf):
        for t in (keys[1], keys[2], values[1], values[2]):
            old = t[page, :, off].clone()
            t[page, :, off] = bad
            again = paged.attend(q, keys, values, table, _i32([300], cuda), scale, q_start=qs, max_q=new)
            t[page, :, off] = old
            assert torch.equal(again[:-1], got[:-1])
            assert not bool(torch.isfinite(again[-1].float()).all())
    assert _status() == 0


@FORMS
def test_pages_that_are_missing(cuda, form, new, H, KVH, D, columns):
    """Ids outside the pool are recorded and their keys left out: what the other keys alone give."""
    import torch
    from locals_b200 import paged

    n = 400
    _, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, n, H, KVH, D, columns, seed=14)
    bad = table.clone()
    gone = [0, 3, 4, 11, 23]
    for i, col in enumerate(gone):
        bad[0, col] = (keys[0].shape[0], -1, 2 ** 31 - 1, -2 ** 31, keys[0].shape[0] + 1)[i]
    got = paged.attend(q, keys, values, bad, _i32([n], cuda), scale, q_start=qs, max_q=new)
    assert _status() == BOUNDS
    # the same in 64 bits: scores of the missing keys are the lowest, by keys that are their queries' opposites
    k, v = R.unpacked(keys), R.unpacked(values)
    G = H // KVH
    ids = table[0, :n // 16].long()
    kb, vb = (x[ids].transpose(0, 1).flatten(1, 2) for x in (k, v))
    s = scale * torch.einsum("ihgd,hjd->hgij", q.double().view(new, KVH, G, D), kb)
    j = torch.arange(n, device=cuda)
    seen = (j[None] <= (n - new + torch.arange(new, device=cuda))[:, None]) & ~torch.isin(j // 16, torch.tensor(gone, device=cuda))[None]
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    ref = torch.einsum("hgij,hjd->ihgd", p, vb).reshape(new, H, D)
    size = torch.einsum("hgij,hjd->ihgd", p, vb.abs()).reshape(new, H, D)
    qk = scale * torch.einsum("ihgd,hjd->hgij", q.double().view(new, KVH, G, D).abs(), kb.abs()).amax(-1)
    moved = 2 * 2.0 ** -11 * qk.permute(2, 0, 1).reshape(new, H, 1)
    assert bool(((got.double() - ref).abs() <= R.U[q.dtype] * ref.abs() + size * (2.0 ** -10 + 2.0 ** -14 + moved) + 2.0 ** -24).all())


@pytest.mark.parametrize("form,new,D,width", [
    (CLUSTERS, 5, 128, 20), (SPLIT, 5, 256, 2000), (TILES, 40, 128, 2000), (TILES, 40, 256, 2000), (DENSE, 140, 128, 2000),
    (DENSE, 140, 256, 2000), (DENSE, 140, 64, 3000)])
def test_lengths_beyond_the_table(cuda, form, new, D, width):
    """Queries whose positions lie beyond the table see the keys that it names (of one page, again and again)."""
    import torch
    from locals_b200 import paged

    _, (q, keys, values, table, qs, scale, _) = _attend(cuda, [new], [160], 8, 2, D, 16, "bfloat16", seed=15, max_q=new)
    assert _forms(1, new, 8, 2, D, width) & form
    wide = table[:, :1].expand(1, width).contiguous()
    beyond = paged.attend(q, keys, values, wide, _i32([16 * width + 5000], cuda), scale, q_start=qs, max_q=new)
    assert _status() == BOUNDS
    # all queries then see all places: 16 keys, as often each
    ref, bound = R.attended(q, keys, values, table[:, :1], _i32([16], cuda), scale, _i32([0, new], cuda), None, 0)
    rows = [paged.attend(q[i:i + 1], keys, values, table[:, :1].contiguous(), _i32([16], cuda), scale) for i in (0, new - 1)]
    assert bool(((beyond[[0, new - 1]].double() - torch.cat(rows).double()).abs()
                 <= 2 * bound[new - 1:].amax() + 2.0 ** -8 * beyond[[0, new - 1]].double().abs()).all())
    again = paged.attend(q, keys, values, wide, _i32([2 ** 31 - 1], cuda), scale, q_start=qs, max_q=new)
    assert bool(torch.isfinite(again).all()) and _status() == BOUNDS
    none = paged.attend(q, keys, values, wide, _i32([-2 ** 31], cuda), scale, q_start=qs, max_q=new)
    assert torch.count_nonzero(none).item() == 0 and _status() == 0


@FORMS
def test_values_of_any_size(cuda, form, new, H, KVH, D, columns):
    from locals_b200 import paged

    _, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, 400, H, KVH, D, columns, seed=12)
    lens = _i32([400], cuda)
    for size in (2.0 ** -16, 2.0 ** 12, 2.0 ** -60, 2.0 ** 60):
        vals = (values[0], values[1] * size, values[2] * size)
        got = paged.attend(q, keys, vals, table, lens, scale, q_start=qs, max_q=new)
        ref, bound = R.attended(q, keys, vals, table, lens, scale, qs, None, 0)
        assert bool(((got.double() - ref).abs() <= bound - 2.0 ** -24 + 2.0 ** -24 * min(size, 1.0)).all()), size


def _sizes(q, keys, values, table, n, scale, window):
    """sum p |v| / sum p of each output, in 64 bits."""
    import torch

    new, H, D = q.shape
    k, v = R.unpacked(keys), R.unpacked(values)
    KVH, page = k.shape[1], k.shape[2]
    ids = table[0, :-(-n // page)].long()
    kb, vb = (x[ids].transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, v))
    s = scale * torch.einsum("ihgd,hjd->hgij", q.double().view(new, KVH, H // KVH, D), kb)
    at, j = (n - new + torch.arange(new, device=q.device))[:, None], torch.arange(n, device=q.device)[None]
    seen = (j <= at) & (j > at - window) if window else j <= at
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    return torch.einsum("hgij,hjd->ihgd", p, vb.abs()).reshape(new, H, D)


def _out_of_sight(cuda, form, new, H, KVH, D, columns, e):
    """Values 2^e of the usual size reach only the rows that see them: the first 64 keys, behind the windows of all queries but
    the first two, and the last token's but one. The others' outputs are those beside ordinary values there, but for the roundings
    of 16-bit operands (2 * 2^-11 of sum p |v|) and outputs, of each."""
    import torch
    from locals_b200 import paged

    n = 6000 if form in (CLUSTERS, SPLIT) else 640  # (several steps a CTA)
    for window, places, rows in ((n - 64 - new + 2, range(64), slice(2, None)), (0, range(n - 2, n - 1), slice(0, -2))):
        plain, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, n, H, KVH, D, columns, seed=31, window=window)
        s, b = values[1].clone(), values[2].clone()
        for j in places:
            at = int(table[0, j // 16]), slice(None), j % 16
            s[at] *= 2.0 ** e
            b[at] *= 2.0 ** e
        got = paged.attend(q, keys, (values[0], s, b), table, _i32([n], cuda), scale, q_start=qs, max_q=new, window=window)
        size = _sizes(q, keys, values, table, n, scale, window)
        bound = 2 * (R.U[q.dtype] * size.clamp(max=plain.double().abs()) + size * (2.0 ** -10 + 2.0 ** -14)) + 2.0 ** -24
        off = ((got.double() - plain.double()).abs() - bound)[rows]
        assert bool((off <= 0).all()), (window, off.max().item())
    assert _status() == 0


@pytest.mark.parametrize("e", [10, 20, 60, 100])
@pytest.mark.parametrize("form,new,H,KVH,D,columns", [x for x in EACH if x[0] in (CLUSTERS, SPLIT)])
def test_large_values_out_of_sight(cuda, form, new, H, KVH, D, columns, e):
    _out_of_sight(cuda, form, new, H, KVH, D, columns, e)


@pytest.mark.parametrize("e", [10, 20, 60, 100])
@pytest.mark.parametrize("form,new,H,KVH,D,columns", [x for x in EACH if x[0] in (TILES, DENSE)])
def test_large_values_out_of_sight_of_many_rows(cuda, form, new, H, KVH, D, columns, e):
    _out_of_sight(cuda, form, new, H, KVH, D, columns, e)


@pytest.mark.parametrize("e", [10, 20, 60, 100])
@FORMS
def test_large_keys_out_of_sight(cuda, form, new, H, KVH, D, columns, e):
    """Keys 2^e of the usual size, as the values of test_large_values_out_of_sight: rows that do not see them answer as beside
    ordinary keys there, but for the roundings of keys (the bound's), probabilities, values and outputs, of each."""
    import torch
    from locals_b200 import paged

    n = 6000 if form in (CLUSTERS, SPLIT) else 640
    for window, places, rows in ((n - 64 - new + 2, range(64), slice(2, None)), (0, range(n - 2, n - 1), slice(0, -2))):
        plain, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, n, H, KVH, D, columns, seed=34, window=window)
        s, b = keys[1].clone(), keys[2].clone()
        for j in places:
            at = int(table[0, j // 16]), slice(None), j % 16
            s[at] *= 2.0 ** e
            b[at] *= 2.0 ** e
        got = paged.attend(q, (keys[0], s, b), values, table, _i32([n], cuda), scale, q_start=qs, max_q=new, window=window)
        ref, bound = R.attended(q, keys, values, table, _i32([n], cuda), scale, qs, None, window)
        off = ((got.double() - ref).abs() - bound)[rows]
        assert bool((off <= 0).all()), (window, off.max().item())
        size = _sizes(q, keys, values, table, n, scale, window)
        near = 2 * (R.U[q.dtype] * size.clamp(max=plain.double().abs()) + size * (2.0 ** -10 + 2.0 ** -14)) + 2.0 ** -24
        # (the roundings of the keys are the same but where one has a power of two of its own: by far most outputs are as near)
        off = ((got.double() - plain.double()).abs() - near)[rows]
        assert (off > 0).double().mean().item() < 0.01
    assert _status() == 0


@FORMS
@pytest.mark.parametrize("what", ["a group of each head", "every 37th token", "all"])
@pytest.mark.parametrize("least", [0.0, 1e-7])
def test_values_of_zero(cuda, form, new, H, KVH, D, columns, what, least):
    """Values that are 0, with scales of 0 or the quantizer's least: heads that fill half of their place, tokens of none."""
    import torch
    from locals_b200 import paged

    n = 500
    _, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, n, H, KVH, D, columns, seed=33)
    w, s, b = (t.clone() for t in values)
    if what == "a group of each head":
        w[..., -8:], s[..., -1], b[..., -1] = 0, least, 0
    else:
        places = range(0, n, 37) if what == "every 37th token" else range(n)
        for j in places:
            at = int(table[0, j // 16]), slice(None), j % 16
            w[at], s[at], b[at] = 0, least, 0
    got = paged.attend(q, keys, (w, s, b), table, _i32([n], cuda), scale, q_start=qs, max_q=new)
    ref, bound = R.attended(q, keys, (w, s, b), table, _i32([n], cuda), scale, qs, None, 0)
    assert bool(((got.double() - ref).abs() <= bound).all())
    if what == "all":
        assert torch.count_nonzero(got).item() == 0
    assert _status() == 0


@FORMS
@pytest.mark.parametrize("least", [0.0, 1e-7])
def test_values_of_one_token(cuda, form, new, H, KVH, D, columns, least):
    """All values are 0 but the first token's: outputs are its weight times its values, however small the weight (to 2^-20 of the
    row's largest; from there 2^-31 of it a value)."""
    import torch
    from locals_b200 import paged

    n = 500
    _, (q, keys, values, table, qs, scale, _) = _one(cuda, form, new, n, H, KVH, D, columns, seed=33)
    w, s, b = (t.clone() for t in values)
    for j in range(1, n):
        at = int(table[0, j // 16]), slice(None), j % 16
        w[at], s[at], b[at] = 0, least, 0
    got = paged.attend(q, keys, (w, s, b), table, _i32([n], cuda), scale, q_start=qs, max_q=new)
    ref, bound = R.attended(q, keys, (w, s, b), table, _i32([n], cuda), scale, qs, None, 0)
    assert bool(((got.double() - ref).abs() <= bound + 2.0 ** -31 * R.unpacked(values).nan_to_num().abs().amax()).all())
    assert _status() == 0
