"""Microscaled 4-bit floating point on the GPU against statements in 64 bits (tests/fp4_reference.py)."""

import pytest

from tests import fp4_reference as R

pytestmark = pytest.mark.gpu

MODES = ["mxfp4", "nvfp4"]


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _dt(name):
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _ok(cuda):
    import torch
    from locals_b200 import kernels

    torch.cuda.synchronize()
    assert kernels.device_status() == 0


def _within(got, want, bound):
    import torch

    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((d / bound).nan_to_num(1e9).max()):.3g} of it"
    assert torch.isfinite(got.double()).all()


def _weights(cuda, g, rows, K, mode, stack=None, spread=4):
    """Random codes with scales around 2^-8, and the values they stand for: (operand, values in 64 bits)."""
    import torch
    from locals_b200 import fp4

    lead = () if stack is None else (stack,)
    codes = torch.randint(0, 16, (*lead, rows, K), generator=g, device=cuda, dtype=torch.int32)
    lo, hi = (119 - spread, 119 + spread) if mode == "mxfp4" else (8, 60)
    byte = torch.randint(lo, hi + 1, (*lead, rows, K // R.GROUP[mode]), generator=g, device=cuda).to(torch.uint8)
    w = codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=cuda, dtype=torch.int32))
    words = w.sum(-1, dtype=torch.int32)
    return fp4.pack(words, byte, mode), R.values(codes, byte, mode, K)


# ---- quantize and dequantize -------------------------------------------------------------------------

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 16), (3, 33), (2, 128), (129, 100), (64, 4096), (5, 1001), (300, 48)])
def test_quantize_is_the_definition(cuda, mode, dtype, scaled, rows, K):
    import torch
    from locals_b200 import fp4

    if scaled and mode == "mxfp4":
        pytest.skip("mxfp4 has no factor")
    g = _gen(cuda, rows * K)
    x = torch.randn((rows, K), generator=g, device=cuda) * torch.exp2(torch.randint(-20, 12, (rows, 1), generator=g, device=cuda).float())
    x[:, ::7] *= 40
    if dtype == "f16":
        x = x.clamp(-6e4, 6e4)
    x = x.to(_dt(dtype))
    f = (x.float().abs().amax() / 2688).reshape(1) if scaled else None
    a = fp4.quantize(x, mode, scale=f)
    codes, byte = R.quantize(x, mode, f)
    _ok(cuda)
    assert a.K == K and a.mode == mode
    n = codes.shape[1]
    assert torch.equal(R.unpack_words(a.codes, n).long(), codes)
    assert not R.unpack_words(a.codes, a.codes.shape[-1] * 8)[:, n:].any()  # zero codes to a multiple of 128
    assert torch.equal(fp4.unpack(a)[1].long(), byte)
    for out in ("f32", dtype):
        want = R.values(codes, byte, mode, K, f)
        got = fp4.dequantize(a, _dt(out))
        # one rounding; with a factor two more in 32 bits before it (2^-24 each)
        tol = 0 if f is None and out == "f32" else R.half_step(_dt(out)) + 2.0 ** -23
        _within(got, want.clamp(-torch.finfo(_dt(out)).max, torch.finfo(_dt(out)).max), tol * want.abs() + torch.finfo(_dt(out)).tiny)


def test_quantize_ties_go_to_the_even_code(cuda):
    import torch
    from locals_b200 import fp4

    v = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6], device=cuda)
    want = [7, 0, 2, 2, 4, 4, 6, 6, 8, 10, 10, 12, 12, 14, 14, 15]
    for mode in MODES:
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            for s in (1.0, 0.25, 8.0):
                a = fp4.quantize((v * s).to(dt)[None].repeat(1, 2), mode)
                assert R.unpack_words(a.codes, 32)[0].tolist() == want * 2, (mode, dt, s)
                assert torch.equal(fp4.dequantize(a, torch.float32)[0, :1], torch.tensor([6 * s], device=cuda))
    # one step above and below each middle, a factor that is no power of two: decided exactly
    f = torch.tensor([0.7310585], device=cuda)
    for k in range(-2, 3):
        x = v.clone()
        x = (x.double() * f.double().item()).float()
        for _ in range(abs(k)):
            x = torch.nextafter(x, torch.full_like(x, float("inf") if k > 0 else float("-inf")))
        a = fp4.quantize(x[None], "nvfp4", scale=f)
        codes, byte = R.quantize(x[None], "nvfp4", f)
        assert torch.equal(R.unpack_words(a.codes, 16).long(), codes) and torch.equal(fp4.unpack(a)[1].long(), byte)
    _ok(cuda)


def test_quantize_edges_of_the_range(cuda):
    import torch
    from locals_b200 import fp4

    inf, nan = float("inf"), float("nan")
    rows = [torch.zeros(64), torch.full((64,), 1e-40), torch.full((64,), 3e38), torch.full((64,), -1.2e-38)]
    for odd in (inf, -inf, nan):
        r = torch.randn(64, generator=torch.Generator().manual_seed(1))
        r[40] = odd
        rows.append(r)
    x = torch.stack(rows).to(cuda)
    for mode in MODES:
        a = fp4.quantize(x, mode)
        codes, byte = R.quantize(x, mode)
        assert torch.equal(fp4.unpack(a)[1].long(), byte), mode
        fine = torch.isfinite(x).unflatten(1, (-1, R.GROUP[mode])).all(-1).repeat_interleave(R.GROUP[mode], 1)
        assert torch.equal(R.unpack_words(a.codes, 64)[fine].long(), codes[fine])
        v = fp4.dequantize(a, torch.float32)
        assert torch.isnan(v[~fine]).all() and torch.isfinite(v[:4]).all() and not v[0].any()
    for f in (1e-45, 1e-30, 1e30, 3e38):  # factors near the ends of the range
        s = torch.tensor([f], device=cuda)
        a = fp4.quantize(x[:4], "nvfp4", scale=s)
        codes, byte = R.quantize(x[:4], "nvfp4", s)
        assert torch.equal(fp4.unpack(a)[1].long(), byte) and torch.equal(R.unpack_words(a.codes, 64).long(), codes), f
    _ok(cuda)


def test_quantize_takes_strides_and_leading_dimensions(cuda):
    import torch
    from locals_b200 import fp4

    x = torch.randn((40, 300), generator=_gen(cuda, 3), device=cuda).to(torch.bfloat16)
    for v in (x[:, 5:201], x[::3, :128], x[:, ::2], x.t(), x[3:4, 1:], x.view(4, 10, 300), x[0], x[:0]):
        a, b = fp4.quantize(v, "nvfp4"), fp4.quantize(v.contiguous().view(-1, v.shape[-1]).clone(), "nvfp4")
        assert torch.equal(a.codes, b.codes) and torch.equal(fp4.unpack(a)[1], fp4.unpack(b)[1])
    _ok(cuda)


# ---- both in 4 bits ------------------------------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 128, 128), (1, 14336, 4096), (2, 130, 96), (15, 257, 288), (16, 129, 2048), (17, 64, 640), (33, 1000, 160),
          (64, 384, 1024), (65, 127, 4096), (128, 2560, 9728), (129, 300, 512), (255, 256, 256), (256, 257, 384), (257, 600, 2048),
          (513, 129, 128), (1000, 2050, 736), (2048, 1024, 4096)]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(cuda, mode, M, N, K):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M + N + K)
    x, xv = _weights(cuda, g, M, K, mode, spread=2)
    w, wv = _weights(cuda, g, N, K, mode)
    want, bound = xv @ wv.T, R.lost(K, xv, wv)
    for out in ("f32", "bf16") + (("f16",) if M < 100 else ()):
        y = fp4.matmul(x, w, dtype=_dt(out))
        _ok(cuda)
        _within(y, want, bound + R.half_step(_dt(out)) * want.abs() + torch.finfo(_dt(out)).tiny)
    assert torch.equal(y, fp4.matmul(x, w, dtype=_dt(out)))  # the same sums in the same order


def test_product_takes_the_matrices_factors(cuda):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 5)
    for M in (3, 40, 300):
        x, w = torch.randn((M, 512), generator=g, device=cuda) * 30, torch.randn((200, 512), generator=g, device=cuda) * 0.002
        fx, fw = ((t.abs().amax() / 2688).reshape(1) for t in (x, w))
        for a, b in ((fx, fw), (None, fw), (fx, None)):
            qx, qw = fp4.quantize(x, "nvfp4", scale=a), fp4.quantize(w, "nvfp4", scale=b)
            xv, wv = fp4.dequantize(qx, torch.float32).double(), fp4.dequantize(qw, torch.float32).double()
            want = xv @ wv.T
            # two factors and their product rounded in 32 bits beside the sum's own losses
            _within(fp4.matmul(qx, qw, dtype=torch.float32), want, R.lost(512, xv, wv) + 2.0 ** -21 * want.abs())
    _ok(cuda)


def test_product_every_scale_counts(cuda):
    """One value of one in each matrix, in every place of a stage and a scale tile: a wrong scale is off by a power of two."""
    import torch
    from locals_b200 import fp4

    for mode in MODES:
        K, M, N = 768, 70, 200
        g = _gen(cuda, 9)
        codes = torch.full((N, K // 8), 0x22222222, dtype=torch.int32, device=cuda)  # ones
        if mode == "mxfp4":
            byte = torch.randint(90, 160, (N, K // 32), generator=g, device=cuda).to(torch.uint8)
        else:
            byte = torch.randint(1, 127, (N, K // 16), generator=g, device=cuda).to(torch.uint8)
        w = fp4.pack(codes, byte, mode)
        k = torch.arange(K, device=cuda)
        for rows in (M, 3 * K):  # a few tokens, and every k
            at = torch.arange(rows, device=cuda) * (11 if rows == M else 1) % K
            x = torch.zeros((rows, K), device=cuda)
            x[torch.arange(rows, device=cuda), at] = 1.0
            qx = fp4.quantize(x, mode)
            y = fp4.matmul(qx, w, dtype=torch.float32)
            want = R.scale_values(byte, mode)[:, (at // R.GROUP[mode])].T
            # 1.0 is 4 * 0.25 in mxfp4 and 6 * 0.171875 in nvfp4: what the operand stands for
            one = fp4.dequantize(qx, torch.float32).double()[torch.arange(rows, device=cuda), at]
            assert torch.equal(y.double(), want * one[:, None]), (mode, rows)
        assert k.numel() == K
    _ok(cuda)


def test_product_leaves_rows_beyond_alone_and_poison_in_other_rows_out(cuda):
    """Rows next to the operands' (not a number) do not reach the result, nor does anything beyond it change."""
    import torch
    from locals_b200 import _lib, fp4
    from locals_b200.kernels import _stream

    for mode in MODES:
        for M, N in ((5, 70), (130, 130), (300, 190)):
            K = 256
            g = _gen(cuda, M)
            x, xv = _weights(cuda, g, M + 128, K, mode, spread=1)
            w, wv = _weights(cuda, g, N + 128, K, mode)
            for t, n in ((x, M), (w, N)):  # scales of the rows behind: not a number
                s = fp4.unpack(t)[1]
                s[n:] = 255 if mode == "mxfp4" else 127
                t.tiles.copy_(fp4.pack(t.codes, s, mode).tiles)
            y = torch.full((M + 3, N), 7.0, device=cuda)
            _lib.call("lq_fp4_qmm", x.codes.data_ptr(), x.tiles.data_ptr(), None, w.codes.data_ptr(), w.tiles.data_ptr(), None, M, N, K,
                      _lib.MXFP4 if mode == "mxfp4" else _lib.NVFP4, 0, _lib.F32, y.data_ptr(), _stream())
            _ok(cuda)
            _within(y[:M], xv[:M] @ wv[:N].T, R.lost(K, xv[:M], wv[:N]) + 1e-30)
            assert (y[M:] == 7.0).all()


def test_a_group_that_is_no_number_makes_its_rows_no_numbers(cuda):
    import torch
    from locals_b200 import fp4

    for mode in MODES:
        x = torch.randn((20, 256), generator=_gen(cuda, 1), device=cuda)
        x[3, 100] = float("inf")
        w = torch.randn((140, 256), generator=_gen(cuda, 2), device=cuda)
        w[130, 7] = float("nan")
        y = fp4.matmul(fp4.quantize(x, mode), fp4.quantize(w, mode), dtype=torch.float32)
        assert torch.isnan(y[3]).all() and torch.isnan(y[:, 130]).all()
        rest = torch.ones_like(y, dtype=torch.bool)
        rest[3], rest[:, 130] = False, False
        assert torch.isfinite(y[rest]).all()
    _ok(cuda)


# ---- 16 bits by 4 ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(cuda, dtype, M, N, K):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M + N + K + 1)
    w, wv = _weights(cuda, g, N, K, "mxfp4")
    x = torch.randn((M, K), generator=g, device=cuda)
    x[:, ::13] *= 25
    x = x.to(_dt(dtype))
    want, bound = R.linear(x, wv, _dt(dtype))
    y = fp4.matmul(x, w)
    _ok(cuda)
    _within(y, want, bound)
    assert torch.equal(y, fp4.matmul(x, w))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_linear_is_exact_where_a_group_spans_13_powers_of_two(cuda, dtype, M):
    """Each row of w picks one value of x (code 1.0, scale 1): the product is that value, in every place."""
    import torch
    from locals_b200 import fp4

    K = 512
    codes = torch.zeros((K, K), dtype=torch.int32, device=cuda)
    codes[torch.arange(K), torch.arange(K)] = 2
    words = (codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=cuda, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    w = fp4.pack(words, torch.full((K, K // 32), 127, dtype=torch.uint8, device=cuda))
    g = _gen(cuda, M)
    e = torch.randint(-13, 1, (M, K), generator=g, device=cuda).float()
    e[:, ::32] = 0
    x = ((1 + torch.rand((M, K), generator=g, device=cuda)) * torch.exp2(e)).to(_dt(dtype))
    x = torch.where(torch.rand((M, K), generator=g, device=cuda) < 0.5, -x, x)
    for s in ((1.0,) if dtype == "f16" else (1.0, 2.0 ** 100, 2.0 ** -90)):
        assert torch.equal(fp4.matmul(x * s, w), x * s)
    small = x.clone()
    small[:, 1::2] *= 2.0 ** -9  # below 2^-13 of the largest: off by at most 2^-21 (fp16: 2^-25) of it
    y = fp4.matmul(small, w)
    most = small.double().abs().unflatten(1, (-1, 32)).amax(-1).repeat_interleave(32, 1)
    _within(y, small.double(), (2.0 ** -21 if dtype == "bf16" else 2.0 ** -25) * most * (1 + 2.0 ** -7) + 1e-9)
    _ok(cuda)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_values_of_every_size_in_different_rows_and_groups(cuda, M):
    """Rows and groups 2^100 apart do not take one another's bits."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M)
    K, N = 640, 150
    w, wv = _weights(cuda, g, N, K, "mxfp4")
    x = torch.randn((M, K), generator=g, device=cuda)
    x = x * torch.exp2(20.0 * (torch.arange(M, device=cuda) % 5 - 2))[:, None].float()
    x = x.to(torch.bfloat16)
    x[:, 64:96] = 0
    want, bound = R.linear(x, wv, torch.bfloat16)
    _within(fp4.matmul(x, w), want, bound)
    x[:, :32] *= 2.0 ** 40  # and a group whose weights are zeros
    codes, s = fp4.unpack(w)
    codes[:, :4] = 0
    want, bound = R.linear(x[:, 32:], wv[:, 32:], torch.bfloat16)
    _within(fp4.matmul(x, fp4.pack(codes, s)), want, bound)
    _ok(cuda)


def test_linear_takes_views_and_refuses_other_formats(cuda):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 4)
    w, _ = _weights(cuda, g, 96, 128, "mxfp4")
    n, _ = _weights(cuda, g, 96, 128, "nvfp4")
    x = torch.randn((24, 400), generator=g, device=cuda).to(torch.float16)
    for v in (x[:, 3:131], x[::2, 8:136], x[:, 1:257:2], x[:, :128].view(4, 6, 128), x[2, 100:228], x[:0, :128], x[:, :128].expand(2, 24, 128)):
        y = fp4.matmul(v, w)
        assert y.shape == (*v.shape[:-1], 96)
        assert torch.equal(y.reshape(-1, 96), fp4.matmul(v.reshape(-1, 128).contiguous().clone(), w))
    q = fp4.quantize(x[:, :128], "mxfp4")
    for bad in (lambda: fp4.matmul(x[:, :128], n), lambda: fp4.matmul(x[:, :96], w), lambda: fp4.matmul(q, n),
                lambda: fp4.matmul(fp4.quantize(x[:, :64]), w), lambda: fp4.matmul(x[:, :128].cpu(), w),
                lambda: fp4.matmul(x[:, :128], w, glu=True) if w.rows % 2 else (_ for _ in ()).throw(ValueError()),
                lambda: fp4.matmul(q, w._replace(tiles=w.tiles[:, :0])), lambda: fp4.matmul(q, w._replace(K=129)),
                lambda: fp4.matmul(q, w._replace(scale=torch.ones(1, device=cuda))), lambda: fp4.quantize(x, "nvfp4", scale=torch.ones(2, device=cuda)),
                lambda: fp4.matmul(x[:, :128], w._replace(codes=w.codes[None], tiles=w.tiles[None])),
                lambda: fp4.grouped(x[:, :128].contiguous(), (torch.zeros(4, device=cuda),) * 5, w, 4)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(TypeError):
        fp4.matmul(x[:, :128].float(), w)
    _ok(cuda)


def test_linear_with_an_infinity_or_no_number_gives_none_in_its_row(cuda):
    import torch
    from locals_b200 import fp4

    w, wv = _weights(cuda, _gen(cuda, 4), 130, 256, "mxfp4")
    for M in (4, 300):
        x = torch.randn((M, 256), generator=_gen(cuda, 5), device=cuda).to(torch.bfloat16)
        x[1, 200], x[2, 0] = float("inf"), float("nan")
        y = fp4.matmul(x, w)
        assert torch.isnan(y[1:3]).all()
        keep = [0, *range(3, M)]
        want, bound = R.linear(x[keep], wv, torch.bfloat16)
        _within(y[keep], want, bound)
    _ok(cuda)


@pytest.mark.parametrize("M,I,K", [(1, 5, 64), (1, 768, 2048), (7, 96, 160), (40, 130, 512), (100, 64, 256), (300, 200, 384)])
def test_glu(cuda, M, I, K):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M + I)
    w, wv = _weights(cuda, g, 2 * I, K, "mxfp4", spread=1)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn((M, K), generator=g, device=cuda).to(dtype)
        want, bound = R.glu(x, wv[0::2], wv[1::2], dtype)
        _within(fp4.matmul(x, w, glu=True), want, bound)
    for mode in MODES:
        x, xv = _weights(cuda, g, M, K, mode, spread=0)
        w, wv = _weights(cuda, g, 2 * I, K, mode, spread=1)
        for out in (torch.bfloat16, torch.float32):
            want, bound = R.glu(xv, wv[0::2], wv[1::2], out)
            _within(fp4.matmul(x, w, dtype=out, glu=True), want, bound)
    _ok(cuda)


# ---- routed experts ---------------------------------------------------------------------------------------

def _experts(cuda, g, E, D, I):
    import torch

    gu, v = _weights(cuda, g, 2 * I, D, "mxfp4", E, 1)
    dn, dv = _weights(cuda, g, D, I, "mxfp4", E, 1)
    return gu, dn, v[:, 0::2], v[:, 1::2], dv, torch


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,E,k,D,I", [
    (1, 8, 2, 256, 96), (1, 64, 4, 2048, 768), (1, 4, 4, 128, 64), (2, 8, 2, 160, 32), (7, 16, 4, 512, 288), (33, 60, 6, 320, 96),
    (64, 64, 4, 2048, 768), (100, 4, 2, 256, 128), (300, 8, 3, 384, 160), (1500, 8, 2, 256, 96), (257, 1, 1, 128, 64)])
def test_experts(cuda, dtype, T, E, k, D, I):
    g = _gen(cuda, T + E)
    gu, dn, gate, up, down, torch = _experts(cuda, g, E, D, I)
    from locals_b200 import fp4, moe

    x = torch.randn((T, D), generator=g, device=cuda).to(_dt(dtype))
    inds = torch.rand((T, E), generator=g, device=cuda).topk(k, -1).indices.to(torch.int32)
    weights = torch.softmax(torch.randn((T, k), generator=g, device=cuda), -1)
    want, bound = R.experts(x, inds, weights, gate, up, down, _dt(dtype))
    y = fp4.experts(x, inds, weights, gu, dn)
    _ok(cuda)
    _within(y, want, bound)
    assert torch.equal(y, fp4.experts(x, inds, weights, gu, dn))
    ys = fp4.switch_glu(x, inds, gu, dn)
    assert ys.shape == (T, k, D)
    _within(moe.combine(ys.reshape(T * k, D), weights, None), want, bound)


def test_experts_that_all_take_one_or_name_one_twice(cuda):
    g = _gen(cuda, 3)
    E, D, I, k = 6, 256, 96, 2
    gu, dn, gate, up, down, torch = _experts(cuda, g, E, D, I)
    from locals_b200 import fp4

    for T in (1, 20, 500):
        x = torch.randn((T, D), generator=g, device=cuda).to(torch.bfloat16)
        weights = torch.rand((T, k), generator=g, device=cuda)
        for inds in (torch.full((T, k), 5), torch.stack([torch.zeros(T), torch.arange(T) % E], 1)):
            inds = inds.to(cuda, torch.int32)
            want, bound = R.experts(x, inds, weights, gate, up, down, torch.bfloat16)
            _within(fp4.experts(x, inds, weights, gu, dn), want, bound)
    empty = fp4.experts(torch.empty((0, D), device=cuda, dtype=torch.bfloat16), torch.empty((0, k), device=cuda, dtype=torch.int32),
                        torch.empty((0, k), device=cuda), gu, dn)
    assert empty.shape == (0, D)
    _ok(cuda)


def test_grouped_leaves_padding_segments_alone(cuda):
    """Pairs of another rank's experts (the padding bucket of group_range) are skipped, their rows left as they were."""
    g = _gen(cuda, 8)
    E, D, N, T, k = 8, 128, 136, 50, 3
    w, wv = _weights(cuda, g, N, D, "mxfp4", 3)
    import torch
    from locals_b200 import _lib, fp4, moe
    from locals_b200.kernels import _stream

    inds = torch.rand((T, E), generator=g, device=cuda).topk(k, -1).indices.to(torch.int32)
    x = torch.randn((T, D), generator=g, device=cuda).to(torch.bfloat16)
    order, starts, experts_, nseg, pos = moe.group_range(inds, 2, 3)
    P = T * k
    out = torch.full((P, N), 5.0, device=cuda, dtype=torch.bfloat16)
    n = _lib.lib().lq_fp4_experts_workspace(P, T, 3, N, D, _lib.BF16)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    _lib.call("lq_fp4_experts", x.data_ptr(), T, order.data_ptr(), k, starts.data_ptr(), experts_.data_ptr(), nseg.data_ptr(), P, T, 0,
              w.codes.data_ptr(), w.tiles.data_ptr(), out.data_ptr(), 3, N, D, _lib.BF16, ws.data_ptr(), n, _stream())
    _ok(cuda)
    flat = inds.reshape(-1)[order.long()].long() - 2
    mine = (flat >= 0) & (flat < 3)
    assert (out[~mine] == 5.0).all()
    xs = x[order.long() // k]
    for e in range(3):
        rows = flat == e
        want, bound = R.linear(xs[rows], wv[e], torch.bfloat16)
        _within(out[rows], want, bound)


def test_experts_out_of_range_are_recorded_and_left_out(cuda):
    import torch
    from locals_b200 import _lib, kernels
    from locals_b200.kernels import _stream

    g = _gen(cuda, 8)
    w, wv = _weights(cuda, g, 64, 128, "mxfp4", 3)
    x = torch.randn((2, 128), generator=g, device=cuda).to(torch.bfloat16)
    out = torch.full((4, 64), 5.0, device=cuda, dtype=torch.bfloat16)
    n = _lib.lib().lq_fp4_experts_workspace(4, 2, 3, 64, 128, _lib.BF16)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    ids = torch.tensor([1, -7, 1 << 20, 2], dtype=torch.int32, device=cuda)
    order = torch.tensor([0, 1, 2, 90], dtype=torch.int32, device=cuda)  # the last names a row that x does not have
    _lib.call("lq_fp4_experts", x.data_ptr(), 2, order.data_ptr(), 2, None, ids.data_ptr(), None, 4, 2, 0, w.codes.data_ptr(),
              w.tiles.data_ptr(), out.data_ptr(), 3, 64, 128, _lib.BF16, ws.data_ptr(), n, _stream())
    torch.cuda.synchronize()
    assert kernels.device_status() == 2  # LQ_DEV_BOUNDS
    assert (out[1:3] == 5.0).all() and not out[3].any()
    want, bound = R.linear(x[:1], wv[1], torch.bfloat16)
    _within(out[:1], want, bound)


# ---- together, in graphs and streams ------------------------------------------------------------------------

def test_a_layer_in_4_bits_and_its_graph(cuda):
    """Norm, experts and a 4-bit MLP as a server runs them: eager, and captured and replayed on new inputs."""
    import torch
    from locals_b200 import fp4, moe, norm

    g = _gen(cuda, 21)
    T, D, I, E, k = 24, 512, 192, 8, 2
    gu, dn, gate, up, down, _ = _experts(cuda, g, E, D, I)
    router = (torch.randn((E, D), generator=g, device=cuda) * 0.05).to(torch.float16)
    layer = fp4.MoELayer(router, gu, dn, k)
    out = fp4.Linear(_weights(cuda, g, D, D, "mxfp4", spread=0)[0])
    wq = fp4.quantize(torch.randn((D, D), generator=g, device=cuda) * 0.05, "nvfp4")
    nw = torch.ones(D, device=cuda, dtype=torch.bfloat16)

    def step(x):
        h, n = norm.add_rms(x, layer(x), nw, 1e-5)
        return fp4.matmul(fp4.quantize(out(n), "nvfp4"), wq), h

    x = torch.randn((T, D), generator=g, device=cuda).to(torch.bfloat16)
    inds, weights = moe.route(x, router, k)
    want, bound = R.experts(x, inds, weights, gate, up, down, torch.bfloat16)
    _within(layer(x), want, bound)
    eager = [t.clone() for t in step(x)]
    static = x.clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(static)
        s.synchronize()
    graphs = []
    for _ in range(2):  # two graphs that share the allocator's pool
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(static)
        graphs.append((gr, res))
    x2 = torch.randn((T, D), generator=g, device=cuda).to(torch.bfloat16)
    eager2 = [t.clone() for t in step(x2)]
    for src, ref in ((x, eager), (x2, eager2), (x, eager)):
        static.copy_(src)
        for gr, res in graphs:
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(res, ref):
                assert torch.equal(a, b)
    _ok(cuda)


def test_two_streams_at_once(cuda):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 2)
    E, D, I = 8, 256, 96
    gu, dn, *_ = _experts(cuda, g, E, D, I)
    w, _v = _weights(cuda, g, 1000, 640, "mxfp4")
    xs = [torch.randn((m, 640), generator=g, device=cuda).to(torch.bfloat16) for m in (1, 40, 300)]
    xe = torch.randn((50, D), generator=g, device=cuda).to(torch.bfloat16)
    inds = torch.rand((50, E), generator=g, device=cuda).topk(2, -1).indices.to(torch.int32)
    wt = torch.rand((50, 2), generator=g, device=cuda)
    want = [fp4.matmul(x, w) for x in xs], fp4.experts(xe, inds, wt, gu, dn)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {0: [], 1: []}
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(([fp4.matmul(x, w) for x in xs], fp4.experts(xe, inds, wt, gu, dn)))
    torch.cuda.synchronize()
    for i in got:
        for a, b in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(a, want[0])) and torch.equal(b, want[1])
    _ok(cuda)


def test_quantized_weights_are_read_after_they_are_written(cuda):
    """Weights quantized right before the product that reads them, over and over in the same place."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 6)
    ws = [torch.randn((2048, 1024), generator=g, device=cuda).to(torch.bfloat16) for _ in range(3)]
    for M in (1, 300):
        x = torch.randn((M, 1024), generator=g, device=cuda).to(torch.bfloat16)
        qx = fp4.quantize(x, "mxfp4")
        torch.cuda.synchronize()
        want = []
        for w in ws:
            q = fp4.quantize(w, "mxfp4")
            torch.cuda.synchronize()
            want.append((fp4.matmul(qx, q), fp4.matmul(x, q)))
            torch.cuda.synchronize()
        got = []
        for i in range(30):
            got.append((fp4.matmul(qx, fp4.quantize(ws[i % 3], "mxfp4")), fp4.matmul(x, fp4.quantize(ws[i % 3], "mxfp4"))))
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(got):
            assert torch.equal(a, want[i % 3][0]) and torch.equal(b, want[i % 3][1])
    _ok(cuda)


def test_offsets_beyond_32_bits(cuda):
    """An output of more than 2^32 bytes, and codes of a matrix of more than 2^31 values."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 6)
    M, N, K = 70001, 32768, 64
    x, xv = _weights(cuda, g, M, K, "mxfp4", spread=1)
    w, wv = _weights(cuda, g, N, K, "mxfp4", spread=1)
    y = fp4.matmul(x, w)
    at = torch.tensor([0, 1, 65535, 65536, M - 1], device=cuda)
    want = xv[at] @ wv.T
    _within(y[at], want, R.lost(K, xv[at], wv) + R.half_step(torch.bfloat16) * want.abs() + 1e-30)
    del y
    big = torch.zeros((300001, 8192), dtype=torch.bfloat16, device=cuda)
    big[-2:] = torch.randn((2, 8192), generator=g, device=cuda).to(torch.bfloat16)
    a = fp4.quantize(big, "nvfp4")
    small = fp4.quantize(big[-2:].clone(), "nvfp4")
    assert torch.equal(a.codes[-2:], small.codes) and not a.codes[:-2].any()
    back = fp4.dequantize(a)
    assert torch.equal(back[-2:], fp4.dequantize(small)) and not back[1000].any()
    _ok(cuda)


# ---- what the experts share with the other formats -------------------------------------------------------------

@pytest.mark.parametrize("P,E", [(2048, 64), (2049, 64), (2049, 1), (5000, 7), (16004, 64), (40000, 1000), (70001, 128)])
def test_group_of_many_pairs(cuda, P, E):
    """Ids grouped in their own order, whatever the number of CTAs."""
    import torch
    from locals_b200 import moe

    g = _gen(cuda, P)
    inds = (torch.rand(P, generator=g, device=cuda) ** 3 * E).long().clamp(max=E - 1)
    inds[P // 2:P // 2 + 300] = E - 1
    for lo, count in ((0, E), (E // 3, max(1, E // 2))):
        if (lo, count) == (0, E):
            order, starts, experts, nseg, pos = moe.group(inds.to(torch.int32), E)
            key = inds
        else:
            order, starts, experts, nseg, pos = moe.group_range(inds.to(torch.int32), lo, count)
            key = torch.where((inds >= lo) & (inds < lo + count), inds - lo, count)
        want = torch.argsort(key, stable=True)
        assert torch.equal(order.long(), want)
        assert torch.equal(pos.long()[want], torch.arange(P, device=cuda))
        ids, counts = torch.unique(key, return_counts=True)
        n = int(nseg)
        assert n == len(ids) and torch.equal(experts[:n].long(), ids)
        assert torch.equal(starts[:n + 1].long(), torch.cat([torch.zeros(1, dtype=torch.long, device=cuda), counts.cumsum(0)]))
    _ok(cuda)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,k,D", [(1, 4, 2048), (3, 1, 8), (77, 6, 136), (33, 2, 100), (500, 8, 264)])
def test_combine_keeps_its_order_of_sums(cuda, dtype, T, k, D):
    """Slots in order in 32 bits, fused multiply and add, rounded once: bit for bit, eight columns a thread or one."""
    import torch
    from locals_b200 import moe

    g = _gen(cuda, T)
    ys = torch.randn((T * k, D), generator=g, device=cuda).to(_dt(dtype))
    w = torch.rand((T, k), generator=g, device=cuda)
    for pos in (None, torch.randperm(T * k, generator=g, device=cuda).to(torch.int32)):
        acc = torch.zeros((T, D), dtype=torch.float32, device=cuda)
        for r in range(k):
            rows = ys[pos.view(T, k)[:, r].long()] if pos is not None else ys.view(T, k, D)[:, r]
            # a product of 8 or 11 bits by 24 and a sum of 24 bits: exact in 64 bits but for its last rounding, then to 32
            acc = (rows.double() * w[:, r, None].double() + acc.double()).float()
        assert torch.equal(moe.combine(ys, w, pos), acc.to(_dt(dtype)))
    _ok(cuda)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 16, 17, 24, 32])
def test_split_sums_of_narrow_tiles_on_two_streams(cuda, dtype, M):
    """Clusters that split K, two CTAs an SM: each has its tensor memory, whatever runs beside it."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M)
    shapes = [(6144, 2560), (4096, 4096), (2048, 768), (14336, 1024)]
    ws = [_weights(cuda, g, n, k, "mxfp4")[0] for n, k in shapes]
    xs = [torch.randn((M, k), generator=g, device=cuda).to(_dt(dtype)) for _, k in shapes]
    want = [fp4.matmul(x, w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(30):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([fp4.matmul(x, w) for x, w in zip(xs, ws)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
    _ok(cuda)
