"""The paged 4-bit cache's operators on the GPU against plain statements in 64 bits (tests/paged_reference.py): block
tables and slot maps, rotary positions with several axes, the cache write and read-back, and attention over the pages."""

import pytest

from tests import paged_reference as R

pytestmark = pytest.mark.gpu

BOUNDS = 2  # LQ_DEV_BOUNDS


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _i32(x, cuda):
    import torch

    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _status():
    from locals_b200 import kernels

    return kernels.device_status()


# ---- plan ------------------------------------------------------------------------------------------

def _run_plan(cuda, cached, new, page, width, free, head, tokens, table=None):
    import torch
    from locals_b200 import paged

    if table is None:
        table = [[1000 + 100 * b + c if c < -(-max(cached[b], 0) // page) else -1 for c in range(width)]
                 for b in range(len(cached))]
    t = _i32(table, cuda)
    f = _i32(free, cuda)
    h = _i32([head], cuda)
    p = paged.plan(_i32(cached, cuda), _i32(new, cuda), t, f, h, page, tokens)
    torch.cuda.synchronize()
    want = R.plan(cached, new, table, free, head, page, tokens)
    got = (t.tolist(), p.lens.tolist(), p.q_start.tolist(), p.positions.tolist(), p.slots.tolist(), p.head.item())
    assert h.item() == head and f.tolist() == free
    return got, want


@pytest.mark.parametrize("cached,new,page,pad", [
    ([0], [1], 16, 0),                       # a first token opens a page
    ([16], [1], 16, 0),                      # the token after a full page
    ([15], [1], 16, 0),                      # the last place of a page
    ([0, 0, 0], [0, 0, 0], 8, 3),            # nothing new, padding only
    ([5, 0, 31, 7], [0, 40, 1, 9], 8, 5),    # a request with nothing new between others
    ([100, 3], [1, 128], 48, 0),             # pages that are no power of two
])
def test_plan(cuda, cached, new, page, pad):
    free = [7 * i % 1009 for i in range(64)]
    got, want = _run_plan(cuda, cached, new, page, 20, free, 3, sum(new) + pad)
    assert got == want
    assert _status() == 0


@pytest.mark.parametrize("B,page,most,seed", [(511, 16, 5, 1), (513, 8, 70, 2), (1500, 32, 3, 3), (8192, 16, 1, 4)])
def test_plan_many_requests(cuda, B, page, most, seed):
    import random

    r = random.Random(seed)
    cached = [r.randrange(0, 200) for _ in range(B)]
    new = [r.randrange(0, most + 1) for _ in range(B)]
    width = -(-(200 + most) // page)
    free = list(range(5000, 5000 + B * width))
    got, want = _run_plan(cuda, cached, new, page, width, free, 11, sum(new) + 7)
    assert got == want
    assert _status() == 0


def test_plan_without_pages_or_columns(cuda):
    # the free list ends within the second request: its last page has no id, its tokens there no slot
    got, want = _run_plan(cuda, [0, 8], [8, 20], 8, 8, [4, 9, 2], 0, 28)
    assert got == want and got[4][-4:] == [-1] * 4
    assert _status() == BOUNDS
    # a table row that is too narrow
    got, want = _run_plan(cuda, [0, 3], [20, 2], 8, 2, list(range(9)), 0, 22)
    assert got == want and got[4][16:20] == [-1] * 4
    assert _status() == BOUNDS
    # negative lengths count as none
    got, want = _run_plan(cuda, [-3, 2], [4, -1], 8, 2, list(range(9)), 0, 4)
    assert got == want
    assert _status() == 0


def test_plan_repeats(cuda):
    """The free list and its head are only read: the same step planned twice gives the same tables."""
    a, _ = _run_plan(cuda, [9, 0], [3, 30], 8, 6, list(range(40, 60)), 5, 33)
    b, _ = _run_plan(cuda, [9, 0], [3, 30], 8, 6, list(range(40, 60)), 5, 33, table=a[0])
    assert a == b


# ---- rotary ----------------------------------------------------------------------------------------

def _rotary_inputs(cuda, N, H, KVH, D, rot, naxes, dtype, seed, far=513):
    import torch
    from locals_b200 import rotary

    g = _gen(cuda, seed)
    dt = getattr(torch, dtype)
    q = (3 * torch.randn((N, H, D), generator=g, device=cuda)).to(dt)
    k = torch.randn((N, KVH, D), generator=g, device=cuda).to(dt) if KVH else None
    cos, sin = rotary.tables(far, rot, 10000.0, cuda)
    pos = torch.randint(0, far, (naxes, N), generator=g, device=cuda, dtype=torch.int32)
    axes = torch.randint(0, naxes, (rot // 2,), generator=g, device=cuda, dtype=torch.int32) if naxes > 1 else None
    return q, k, pos, cos, sin, axes


def _check_rotated(got, x, pos, cos, sin, axes, inter):
    ref, slack = R.rotated(x, pos, cos, sin, axes, inter)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert bool(((got.double() - ref).abs() <= R.U[x.dtype] * ref.abs() + slack + 2.0 ** -24).all())
    rot = 2 * cos.shape[1]
    import torch

    assert torch.equal(got[..., rot:], x[..., rot:])
    assert torch.equal(got, R.rotated32(x, pos, cos, sin, axes, inter).to(x.dtype))


@pytest.mark.parametrize("N,H,KVH,D,rot,naxes,inter,dtype", [
    (1, 32, 8, 128, 128, 3, False, "bfloat16"),
    (3, 4, 1, 128, 128, 1, True, "float16"),
    (257, 3, 2, 80, 80, 2, False, "float16"),     # halves of 40
    (5, 2, 0, 72, 72, 2, False, "bfloat16"),      # halves of 36: 8-byte pieces
    (7, 1, 1, 96, 24, 3, False, "bfloat16"),      # halves of 12, most of the row copied
    (9, 2, 1, 64, 6, 2, False, "float16"),        # halves of 3: one value at a time
    (9, 2, 1, 64, 6, 3, True, "bfloat16"),
    (4001, 16, 16, 64, 32, 2, True, "bfloat16"),  # several rows a thread
    (2049, 12, 4, 256, 64, 1, False, "float16"),
])
def test_rotary(cuda, N, H, KVH, D, rot, naxes, inter, dtype):
    from locals_b200 import rotary

    q, k, pos, cos, sin, axes = _rotary_inputs(cuda, N, H, KVH, D, rot, naxes, dtype, N + D)
    qo, ko = rotary.rotate(q, k, pos, cos, sin, axes, interleaved=inter)
    _check_rotated(qo, q, pos, cos, sin, axes, inter)
    if KVH:
        _check_rotated(ko, k, pos, cos, sin, axes, inter)
    else:
        assert ko is None
    assert _status() == 0


def test_rotary_strides_and_sections(cuda):
    """q and k as slices of one fused projection, odd offsets, positions (N,), sections of axes, and no tokens."""
    import torch
    from locals_b200 import rotary

    N, H, KVH, D = 37, 4, 2, 64
    g = _gen(cuda, 5)
    for off in (0, 1, 4):
        qkv = torch.randn((N, (H + 2 * KVH) * D + 8), generator=g, device=cuda).to(torch.bfloat16)
        q = qkv[:, off:off + H * D].view(N, H, D)
        k = qkv[:, H * D + off:H * D + off + KVH * D].view(N, KVH, D)
        cos, sin = rotary.tables(100, D, 500000.0, cuda)
        pos = torch.arange(N, dtype=torch.int32, device=cuda)
        qo, ko = rotary.rotate(q, k, pos, cos, sin)
        _check_rotated(qo, q.contiguous(), pos, cos, sin, None, False)
        _check_rotated(ko, k.contiguous(), pos, cos, sin, None, False)
    axes = rotary.sections((8, 12, 12), cuda)
    pos = torch.stack([pos, 2 * pos, pos * 0])
    qo, ko = rotary.rotate(q, None, pos, cos, sin, axes)
    _check_rotated(qo, q.contiguous(), pos, cos, sin, axes, False)
    empty, _ = rotary.rotate(q[:0], None, pos[:, :0].contiguous(), cos, sin, axes)
    assert empty.shape == (0, H, D)
    assert _status() == 0


def test_rotary_position_outside_the_tables(cuda):
    import torch
    from locals_b200 import rotary

    q, k, pos, cos, sin, _ = _rotary_inputs(cuda, 5, 2, 1, 64, 64, 1, "bfloat16", 3, far=10)
    pos[0, 1], pos[0, 3] = 10, -1
    qo, _ = rotary.rotate(q, k, pos, cos, sin)
    ref, _ = rotary.rotate(q, k, pos.clamp(0, 9), cos, sin)
    assert torch.equal(qo, ref)
    assert _status() == BOUNDS


# ---- append and read -------------------------------------------------------------------------------

@pytest.mark.parametrize("N,H,KVH,D,rot,naxes,inter,page,dtype", [
    (1, 32, 8, 128, 128, 3, False, 16, "bfloat16"),
    (67, 8, 4, 128, 64, 2, False, 8, "bfloat16"),
    (130, 3, 1, 64, 64, 1, True, 24, "float16"),
    (33, 4, 2, 256, 64, 3, False, 32, "float16"),
    (19, 0, 3, 64, 16, 2, True, 16, "bfloat16"),
    (1030, 5, 5, 256, 256, 1, False, 64, "bfloat16"),
])
def test_append(cuda, N, H, KVH, D, rot, naxes, inter, page, dtype):
    import torch
    from locals_b200 import kernels, paged

    q, k, pos, cos, sin, axes = _rotary_inputs(cuda, N, max(H, 1), KVH, D, rot, naxes, dtype, N)
    g = _gen(cuda, N + 1)
    v = torch.randn((N, KVH, D), generator=g, device=cuda).to(k.dtype)
    v[:, :, 3] *= 20  # an outlier channel
    v[0] = 0          # a constant group
    pages = 2 * (-(-N // page)) + 1
    keys, values = paged.pool(pages, KVH, page, D, k.dtype, cuda)
    for t in (*keys, *values):
        t.fill_(1)
    before = [t.clone() for t in (*keys, *values)]
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:N].to(torch.int32)
    if N > 4:
        slots[2] = -1
    qo = paged.append(q if H else None, k, v, slots, keys, values, pos, cos, sin, axes, interleaved=inter)
    if H:
        _check_rotated(qo, q, pos, cos, sin, axes, inter)
    else:
        assert qo is None
    live = slots >= 0
    at = (slots[live] // page).long(), (slots[live] % page).long()
    krot = R.rotated32(k, pos, cos, sin, axes, inter)
    exact, _ = R.rotated(k, pos, cos, sin, axes, inter)
    rk, rv = paged.read(keys, values, slots)
    for triple, x32, x64, back in ((keys, krot, exact, rk), (values, v.float(), v.double(), rv)):
        # the codes, scales and biases of the library's quantizer on the 32-bit values
        wq, s, b = kernels.quantize(x32[live].reshape(-1, D).contiguous(), bits=4, dtype=k.dtype)
        n = int(live.sum())
        assert torch.equal(triple[0][at[0], :, at[1]], wq.view(n, KVH, -1))
        assert torch.equal(triple[1][at[0], :, at[1]], s.view(n, KVH, -1))
        assert torch.equal(triple[2][at[0], :, at[1]], b.view(n, KVH, -1))
        assert torch.equal(back[live], kernels.dequantize(wq, s, b, bits=4).view(n, KVH, D))
        assert torch.count_nonzero(back[~live]) == 0
        # 15 steps cover the group's range up to one step, and the scale and bias are rounded to the dtype
        grp = x64[live].unflatten(-1, (-1, 64))
        step = (grp.amax(-1) - grp.amin(-1)) / 15
        off = (R.unpacked((triple[0][at[0], :, at[1]], triple[1][at[0], :, at[1]], triple[2][at[0], :, at[1]]))
               - x64[live]).unflatten(-1, (-1, 64)).abs().amax(-1)
        u = R.U[k.dtype]
        assert bool((off <= 1.001 * step + u * (15 * 1.07 * step + grp.abs().amax(-1)) + 2e-6).all())
    # nothing else in the pool changed
    mask = torch.ones((pages, page), dtype=torch.bool, device=cuda)
    mask[at] = False
    for t, old in zip((*keys, *values), before):
        assert torch.equal(t.transpose(1, 2)[mask], old.transpose(1, 2)[mask])
    assert _status() == 0


def test_append_without_rotation_and_out_of_range(cuda):
    import torch
    from locals_b200 import kernels, paged

    g = _gen(cuda, 2)
    qkv = torch.randn((6, 8, 128), generator=g, device=cuda).to(torch.bfloat16)
    k, v = qkv[:, 4:6], qkv[:, 6:8]  # slices of one fused projection
    keys, values = paged.pool(2, 2, 8, 128, torch.bfloat16, cuda)
    slots = _i32([3, 15, 16, -1, 2 ** 31 - 1, 0], cuda)  # 16 and beyond lie outside the pool
    qo = paged.append(qkv[:, :4], k, v, slots, keys, values)
    assert torch.equal(qo, qkv[:, :4])
    assert _status() == BOUNDS
    ok = _i32([3, 15, 0], cuda)
    rk, rv = paged.read(keys, values, ok)
    for back, x in ((rk, k), (rv, v)):
        x = x[[0, 1, 5]].contiguous()
        assert torch.equal(back, kernels.dequantize(*kernels.quantize(x.view(-1, 128), bits=4), bits=4).view_as(x))
    assert int((keys[1] != 0).any(-1).sum()) == 6  # three tokens of two heads, nothing else
    assert _status() == 0


# ---- attend ----------------------------------------------------------------------------------------

def _cache(cuda, lens, KVH, D, page, dtype, seed, extra=3):
    """A pool whose unused rows hold NaN scales and whose unused table entries are -1."""
    import torch
    from locals_b200 import kernels

    g = _gen(cuda, seed)
    dt = getattr(torch, dtype)
    B = len(lens)
    width = max(1, max(-(-n // page) for n in lens)) + 1
    used = [-(-n // page) for n in lens]
    pages = sum(used) + extra
    ids = torch.randperm(pages, generator=g, device=cuda).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=cuda)
    live = torch.zeros((pages, page), dtype=torch.bool, device=cuda)
    at = 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = ids[at:at + used[b]]
        for j in range(used[b]):
            live[ids[at + j].long(), :min(page, n - j * page)] = True
        at += used[b]
    out = []
    for spread in (2.0, 1.0):
        x = torch.randn((pages, KVH, page, D), generator=g, device=cuda) * spread
        x[..., 5] *= 4
        wq, s, b = kernels.quantize(x.view(-1, D).contiguous(), bits=4, dtype=dt)
        s, b = s.view(pages, KVH, page, -1), b.view(pages, KVH, page, -1)
        dead = ~live[:, None, :, None].expand_as(s)
        out.append((wq.view(pages, KVH, page, -1), s.masked_fill(dead, float("nan")).contiguous(),
                    b.masked_fill(dead, float("nan")).contiguous()))
    return out[0], out[1], table


def _attend(cuda, new, lens, H, KVH, D, page, dtype, window=0, sinks=False, seed=0, scale=None, pad=0, max_q=None, columns=0):
    import torch
    from locals_b200 import paged

    g = _gen(cuda, seed + 77)
    keys, values, table = _cache(cuda, lens, KVH, D, page, dtype, seed)
    if columns:  # room for more than the requests have
        table = torch.cat([table, torch.full((len(lens), columns), -1, dtype=torch.int32, device=cuda)], 1)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    one = all(n == 1 for n in new) and not pad and max_q is None
    q = (1.5 * torch.randn((start[-1] + pad, H, D), generator=g, device=cuda)).to(getattr(torch, dtype))
    sk = 2 * torch.randn((H,), generator=g, device=cuda) if sinks else None
    qs = _i32(start, cuda)
    scale = D ** -0.5 if scale is None else scale
    got = paged.attend(q, keys, values, table, _i32(lens, cuda), scale, q_start=None if one else qs,
                       max_q=1 if one else (max_q or max(1, *new)), sinks=sk, window=window)
    ref, bound = R.attended(q[:start[-1]], keys, values, table, _i32(lens, cuda), scale, qs, sk, window)
    assert bool(torch.isfinite(got).all())
    off = (got[:start[-1]].double() - ref).abs() - bound
    assert bool((off <= 0).all()), f"beyond the bound by {off.max().item()}"
    assert torch.count_nonzero(got[start[-1]:]).item() == 0
    assert _status() == 0
    return got, (q, keys, values, table, qs, scale, sk)


@pytest.mark.parametrize("lens,H,KVH,D,page,dtype,window,sinks", [
    ([1], 32, 8, 128, 16, "bfloat16", 0, False),             # one key
    ([1, 8, 9, 16, 17], 8, 8, 128, 8, "float16", 0, False),  # one query head a kv head; around the page's end
    ([333, 64, 65, 127, 128, 129], 12, 4, 128, 24, "bfloat16", 0, True),
    ([700, 31], 16, 1, 64, 16, "float16", 0, False),         # 16 query heads on one kv head
    ([515, 2], 10, 2, 256, 32, "bfloat16", 0, True),
    ([2049], 64, 4, 128, 48, "bfloat16", 0, False),
    ([300, 40, 1], 8, 2, 64, 16, "bfloat16", 33, True),      # a window
    ([300, 40, 1], 8, 2, 128, 16, "float16", 1, False),      # a window of the query itself
    ([20000], 32, 4, 128, 16, "bfloat16", 0, False),         # split over many blocks and joined
    ([20000, 5, 131, 9000], 4, 2, 256, 16, "float16", 0, True),
    ([777], 20, 1, 128, 16, "bfloat16", 0, False),           # 20 query heads a kv head
])
def test_attend_one_token(cuda, lens, H, KVH, D, page, dtype, window, sinks):
    _attend(cuda, [1] * len(lens), lens, H, KVH, D, page, dtype, window, sinks, seed=sum(lens))


@pytest.mark.parametrize("new,lens,H,KVH,D,page,dtype,window,sinks", [
    ([2, 1], [2, 50], 8, 4, 128, 16, "bfloat16", 0, False),
    ([5, 3, 4], [400, 3, 129], 16, 2, 256, 32, "bfloat16", 0, False),  # drafts; a request of new tokens only
    ([3, 0, 4], [70, 90, 4], 8, 8, 64, 8, "float16", 0, True),         # a request with nothing new
    ([7], [1000], 6, 2, 128, 16, "float16", 100, False),
    ([33], [33], 4, 4, 128, 16, "bfloat16", 0, False),                 # a prompt of its own
    ([130, 1, 64], [190, 500, 64], 8, 2, 128, 16, "bfloat16", 0, True),  # prompts and decoding in one batch
    ([257], [300], 5, 1, 64, 24, "float16", 0, False),
    ([129], [640], 4, 2, 256, 16, "bfloat16", 50, False),
    ([200, 1, 1], [1500, 1, 2000], 16, 2, 128, 64, "float16", 0, True),
])
def test_attend_several_tokens(cuda, new, lens, H, KVH, D, page, dtype, window, sinks):
    _attend(cuda, new, lens, H, KVH, D, page, dtype, window, sinks, seed=sum(lens) + 1)


def test_attend_nothing_to_see(cuda):
    """Requests without a key (0, sink or not), padding rows past the last query, and a batch of no queries."""
    import torch
    from locals_b200 import paged

    for sinks in (False, True):
        got, _ = _attend(cuda, [1, 1, 1], [0, 5, 0], 8, 2, 128, 16, "bfloat16", 0, sinks, seed=4, pad=3)
        assert torch.count_nonzero(got[0]).item() == 0 and torch.count_nonzero(got[2]).item() == 0
    got, (q, keys, values, table, qs, scale, _) = _attend(cuda, [40, 1], [40, 7], 8, 2, 128, 16, "float16", seed=5,
                                                          pad=100)
    assert paged.attend(q[:0], keys, values, table, _i32([40, 7], cuda), scale, q_start=qs, max_q=1).shape == (0, 8, 128)
    none = paged.attend(q[:2], keys, values, table, _i32([40, 7], cuda), scale, q_start=_i32([0, 0, 0], cuda), max_q=4)
    assert torch.count_nonzero(none).item() == 0


def test_attend_extremes(cuda):
    """Scores far apart (one key takes all), equal scores, sinks of +-infinity, and a scale of 0 or below."""
    import torch
    from locals_b200 import paged

    for scale in (40.0, 0.0, -1.0):
        _attend(cuda, [1, 1], [300, 65], 8, 2, 128, 16, "bfloat16", seed=6, scale=scale)
        _attend(cuda, [40], [300], 8, 2, 128, 16, "float16", seed=7, scale=scale)
    _, (q, keys, values, table, qs, scale, _) = _attend(cuda, [1], [300], 8, 2, 128, 16, "bfloat16", seed=8)
    lens = _i32([300], cuda)
    plain = paged.attend(q, keys, values, table, lens, scale)
    low = torch.full((8,), -float("inf"), device=cuda)
    assert torch.equal(paged.attend(q, keys, values, table, lens, scale, sinks=low), plain)
    assert torch.equal(paged.attend(q, keys, values, table, lens, scale, sinks=torch.full_like(low, -3e38)), plain)
    high = torch.full((8,), 3e38, device=cuda)
    assert torch.count_nonzero(paged.attend(q, keys, values, table, lens, scale, sinks=high)).item() == 0


def test_attend_masked_places_may_hold_anything(cuda):
    """A later token of infinite or NaN scale changes no earlier query of the same request."""
    import torch
    from locals_b200 import paged

    for new, n in ((4, 50), (40, 300)):
        got, (q, keys, values, table, qs, scale, _) = _attend(cuda, [new], [n], 8, 2, 128, 16, "bfloat16", seed=9 + new)
        last = int(table[0, (n - 1) // 16]), (n - 1) % 16
        for bad in (float("nan"), float("inf")):
            for t in (values[1], values[2], keys[2]):
                old = t[last[0], :, last[1]].clone()
                t[last[0], :, last[1]] = bad
                again = paged.attend(q, keys, values, table, _i32([n], cuda), scale, q_start=qs, max_q=new)
                t[last[0], :, last[1]] = old
                assert torch.equal(again[:-1], got[:-1])
                assert not bool(torch.isfinite(again[-1].float()).all())


def test_attend_values_of_any_size(cuda):
    """Values (and their scales) of 2^-16 to 2^12 of the usual size, and both in one request."""
    import torch
    from locals_b200 import paged

    for new in (1, 40):
        _, (q, keys, values, table, qs, scale, _) = _attend(cuda, [new], [400], 8, 2, 128, 16, "bfloat16", seed=12)
        lens = _i32([400], cuda)
        for size in (2.0 ** -16, 2.0 ** 12):
            vals = (values[0], values[1] * size, values[2] * size)
            got = paged.attend(q, keys, vals, table, lens, scale, q_start=qs, max_q=new)
            ref, bound = R.attended(q, keys, vals, table, lens, scale, qs, None, 0)
            # (values that fall below 2^-14 may be held as 16-bit subnormals: 2^-25 more a value)
            assert bool(((got.double() - ref).abs() <= bound + 2.0 ** -24).all())
        mixed = [t.clone() for t in values[1:]]
        for t in mixed:
            t[:, :, ::2] *= 2.0 ** 9
        vals = (values[0], *mixed)
        got = paged.attend(q, keys, vals, table, lens, scale, q_start=qs, max_q=new)
        ref, bound = R.attended(q, keys, vals, table, lens, scale, qs, None, 0)
        assert bool(((got.double() - ref).abs() <= bound).all())


def test_attend_table_and_pages_out_of_range(cuda):
    """A length beyond the table and page ids outside the pool are recorded, and their keys left out."""
    import torch
    from locals_b200 import paged

    for new in (1, 40):
        _, (q, keys, values, table, qs, scale, _) = _attend(cuda, [new], [160], 8, 2, 128, 16, "bfloat16", seed=14)
        bad = table.clone()
        bad[0, 3], bad[0, 4] = keys[0].shape[0], -1
        got = paged.attend(q, keys, values, bad, _i32([160], cuda), scale, q_start=qs, max_q=new)
        assert bool(torch.isfinite(got).all())
        assert _status() == BOUNDS
        got = paged.attend(q, keys, values, table[:, :8].contiguous(), _i32([160], cuda), scale, q_start=qs, max_q=new)
        assert bool(torch.isfinite(got).all())
        assert _status() == BOUNDS


def test_attend_repeats_and_streams(cuda):
    """The same call gives the same bits, on another stream too, and inside a CUDA graph."""
    import torch
    from locals_b200 import paged

    for new, lens in (([1, 1, 1], [9000, 3, 511]), ([70, 1, 5], [900, 4000, 6])):
        got, (q, keys, values, table, qs, scale, _) = _attend(cuda, new, lens, 16, 2, 128, 16, "bfloat16", seed=15)
        ln = _i32(lens, cuda)
        args = dict(q_start=qs, max_q=max(new))
        first = paged.attend(q, keys, values, table, ln, scale, **args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = paged.attend(q, keys, values, table, ln, scale, **args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            third = paged.attend(q, keys, values, table, ln, scale, **args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, second) and torch.equal(first, third) and torch.equal(first, got)


def test_step_of_a_batch(cuda):
    """Plan, append and attend together, prompt then decode, against attention over the unpacked cache."""
    import torch
    from locals_b200 import paged, rotary

    B, H, KVH, D, page, width = 3, 8, 2, 128, 16, 8
    g = _gen(cuda, 21)
    keys, values = paged.pool(32, KVH, page, D, torch.bfloat16, cuda)
    table = torch.full((B, width), -1, dtype=torch.int32, device=cuda)
    free = torch.randperm(32, generator=g, device=cuda).to(torch.int32)
    head = torch.zeros(1, dtype=torch.int32, device=cuda)
    cached = torch.zeros(B, dtype=torch.int32, device=cuda)
    cos, sin = rotary.tables(256, D, device=cuda)
    for new in ([50, 3, 17], [1, 1, 1], [1, 0, 4]):
        tokens = sum(new)
        nw = _i32(new, cuda)
        p = paged.plan(cached, nw, table, free, head, page, tokens)
        q, k, v = (torch.randn((tokens, h, D), generator=g, device=cuda).to(torch.bfloat16) for h in (H, KVH, KVH))
        qr = paged.append(q, k, v, p.slots, keys, values, p.positions, cos, sin)
        got = paged.attend(qr, keys, values, table, p.lens, D ** -0.5, q_start=p.q_start, max_q=max(new))
        ref, bound = R.attended(qr, keys, values, table, p.lens, D ** -0.5, p.q_start, None, 0)
        assert bool(((got.double() - ref).abs() <= bound).all())
        cached, head = p.lens, p.head
    assert cached.tolist() == [52, 4, 22] and head.item() == 4 + 1 + 2
    assert _status() == 0


def test_queries_keys_and_values_on_any_boundary(cuda):
    """Slices whose rows start 2 bytes past a boundary, or lie an odd number of values apart, give what copies give."""
    import torch
    from locals_b200 import paged, rotary

    g = _gen(cuda, 31)
    N, H, KVH, D, page = 5, 4, 2, 64, 8
    cos, sin = rotary.tables(64, D, device=cuda)
    pos = torch.arange(N, dtype=torch.int32, device=cuda)
    slots = _i32([0, 9, 3, 12, 5], cuda)
    for width, off in (((H + 2 * KVH) * D + 1, 1), ((H + 2 * KVH) * D + 8, 3)):
        qkv = torch.randn((N, width), generator=g, device=cuda).to(torch.bfloat16)
        q, k, v = (qkv[:, off + a * D:off + (a + h) * D].view(N, h, D) for a, h in ((0, H), (H, KVH), (H + KVH, KVH)))
        for inter in (False, True):
            caches = [paged.pool(3, KVH, page, D, torch.bfloat16, cuda) for _ in range(2)]
            a = paged.append(q, k, v, slots, *caches[0], pos, cos, sin, interleaved=inter)
            b = paged.append(q.contiguous(), k.contiguous(), v.contiguous(), slots, *caches[1], pos, cos, sin,
                             interleaved=inter)
            assert torch.equal(a, b)
            for x, y in zip((*caches[0][0], *caches[0][1]), (*caches[1][0], *caches[1][1])):
                assert torch.equal(x, y)
            for x, y in zip(rotary.rotate(q, k, pos, cos, sin, interleaved=inter),
                            rotary.rotate(q.contiguous(), k.contiguous(), pos, cos, sin, interleaved=inter)):
                assert torch.equal(x, y)
        table = _i32([[0, 1], [1, 0], [2, 1], [0, 2], [1, 2]], cuda)
        lens = _i32([9, 3, 16, 1, 8], cuda)
        keys, values = caches[0]
        assert torch.equal(paged.attend(q, keys, values, table, lens, 0.1),
                           paged.attend(q.contiguous(), keys, values, table, lens, 0.1))


def test_attend_on_the_other_side_of_each_rule(cuda):
    """Lengths, batches and rows at which another form takes over: clusters of 8 to 1 CTAs, the even split, tiles unpacked
    in place and unpacked first."""
    _attend(cuda, [1], [900], 4, 1, 128, 16, "bfloat16", seed=40)              # one cluster of 8
    _attend(cuda, [1] * 70, [130 + 7 * i for i in range(70)], 8, 2, 64, 16, "float16", seed=41)   # clusters of fewer
    _attend(cuda, [1] * 130, [3 * i + 1 for i in range(130)], 4, 4, 64, 8, "bfloat16", seed=42)   # more items than CTAs
    _attend(cuda, [2, 2], [9000, 12], 16, 2, 128, 32, "bfloat16", seed=43)     # 16 rows, the even split
    _attend(cuda, [64, 3], [200, 3000], 8, 1, 128, 16, "float16", seed=44)     # two tiles of rows: unpacked in place
    _attend(cuda, [65, 3], [200, 3000], 8, 1, 128, 16, "float16", seed=45)     # a third: unpacked first
    _attend(cuda, [300, 1, 40], [700, 600, 41], 3, 1, 256, 24, "bfloat16", 0, True, seed=46)


@pytest.mark.parametrize("new,lens,H,KVH,D,page,dtype,window,sinks", [
    ([3, 2, 1, 3], [5, 700, 1, 131], 8, 1, 128, 16, "bfloat16", 0, True),       # 24 rows: two tiles, cut within a query's heads
    ([7] * 40, [7 + 61 * i for i in range(40)], 9, 3, 64, 8, "float16", 0, False),  # 21 rows of 3 heads
    ([2, 1], [40, 9000], 64, 4, 128, 32, "bfloat16", 100, False),               # 32 rows, a window, clusters
    ([5, 0, 4], [2000, 30, 6000], 12, 2, 64, 16, "float16", 777, True),         # 30 rows; a request without queries
    ([1] * 3, [300, 17, 5000], 32, 1, 128, 16, "float16", 0, True),             # one query of 32 heads
    ([3, 3], [2500, 3], 8, 1, 256, 16, "bfloat16", 0, False),                   # 24 rows at 256 dimensions
])
def test_attend_two_tiles_of_rows(cuda, new, lens, H, KVH, D, page, dtype, window, sinks):
    _attend(cuda, new, lens, H, KVH, D, page, dtype, window, sinks, seed=50)


@pytest.mark.parametrize("new,lens,H,KVH,D,page,dtype,window,sinks", [
    ([8, 5], [1000, 64], 16, 2, 128, 16, "bfloat16", 0, False),      # 64 rows: four tiles
    ([9, 5], [1000, 64], 16, 2, 128, 16, "bfloat16", 0, False),      # 72: unpacked to tiles in place
    ([16] * 9, [16 + 400 * i for i in range(9)], 4, 1, 64, 8, "float16", 300, True),
    ([5, 1], [3000, 2], 8, 1, 256, 32, "float16", 0, True),          # 40 rows at 256 dimensions, in place
])
def test_attend_on_both_sides_of_the_row_limit(cuda, new, lens, H, KVH, D, page, dtype, window, sinks):
    _attend(cuda, new, lens, H, KVH, D, page, dtype, window, sinks, seed=60)


@pytest.mark.parametrize("new,lens,H,KVH,D,page,dtype,window,sinks", [
    ([33], [33], 16, 4, 128, 16, "bfloat16", 0, False),                  # one tile of rows
    ([130, 1, 64], [190, 500, 64], 8, 2, 128, 16, "bfloat16", 0, True),  # three tiles; prompts and decoding in one batch
    ([257], [300], 5, 1, 64, 24, "float16", 0, False),                   # six tiles
    ([60, 33], [1000, 35], 12, 2, 64, 8, "float16", 77, True),           # two tiles, windows
    ([129], [640], 4, 2, 256, 16, "bfloat16", 50, False),
    ([30, 0, 9], [30, 9, 2000], 8, 1, 256, 32, "float16", 0, True),      # a request without queries
    ([200, 1, 1], [1500, 1, 2000], 16, 2, 128, 64, "float16", 0, True),
])
@pytest.mark.parametrize("room", [130_000, 2_400_000])
def test_attend_in_a_wide_table(cuda, new, lens, H, KVH, D, page, dtype, window, sinks, room):
    """Tables with room for long contexts: requests of many rows are taken in tiles of 128 and 256 rows, their keys unpacked
    first, or, where all that the table can name would not fit the workspace as fp16, tile by tile."""
    _attend(cuda, new, lens, H, KVH, D, page, dtype, window, sinks, seed=70, columns=room // page)


@pytest.mark.parametrize("most", [51, 101])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attend_prompts_at_256_dimensions(cuda, dtype, most):
    """Many items of few steps a CTA: every warp has to have its row's last product before it writes the row."""
    import torch

    new = [most, 1, most - 20, 1, most, 30, 1, most // 2, 1, most - 1, 1]
    lens = [144, 623, 2692, 592, 565, 909, 659, 119, 1495, 803, 1523]
    for seed in (80, 81):
        got, (q, keys, values, table, qs, scale, sk) = _attend(cuda, new, lens, 5, 1, 256, 16, dtype, seed=seed, columns=4000)
        from locals_b200 import paged
        for _ in range(5):
            again = paged.attend(q, keys, values, table, _i32(lens, cuda), scale, q_start=qs, max_q=max(new))
            assert torch.equal(got, again)
