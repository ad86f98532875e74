"""Microscaled 4-bit floating point on the GPU, where a call could go wrong: against statements in 64 bits."""

import pytest

from tests import fp4_reference as R

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _dt(name):
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _status(cuda):
    import torch
    from locals_b200 import kernels

    torch.cuda.synchronize()
    return kernels.device_status()


def _stack(cuda, g, E, rows, K, size=1.0):
    """A stack of E random mxfp4 matrices, any K: (operand, values in 64 bits)."""
    import torch
    from locals_b200 import fp4

    parts = [fp4.quantize(torch.randn((rows, K), generator=g, device=cuda) * size, "mxfp4") for _ in range(E)]
    w = fp4.Fp4(torch.stack([p.codes for p in parts]), torch.stack([p.tiles for p in parts]), "mxfp4", K)
    return w, torch.stack([fp4.dequantize(p, torch.float32).double() for p in parts])


def _experts(x, inds, weights, gate_up, down):
    """The routed experts in 64 bits; ids outside the stack contribute nothing."""
    import torch

    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(gate_up.shape[0]):
        t, slot = torch.where(inds == e)
        gu = x[t].double() @ gate_up[e].T
        h = torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]
        y.index_add_(0, t, weights[t, slot, None].double() * (h @ down[e].T))
    return y


def _rms(t):
    return float(t.double().square().mean().sqrt())


# ---- routed experts ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,E,k,D,I", [(1, 8, 4, 256, 96), (1, 4, 2, 101, 37), (2, 8, 2, 160, 33), (20, 6, 2, 130, 64), (40, 2, 2, 254, 72),
                                       (64, 16, 4, 256, 192), (300, 4, 2, 256, 130), (900, 2, 1, 64, 66)])
def test_experts_are_rounded_once(cuda, dtype, T, E, k, D, I):
    """y is off by little more than its own rounding. What else there is adds in squares: the hidden rows' pieces (2^-14 of a value
    at most, where half a step is 2^-9 or 2^-12), sums in 32 bits (some 24 steps of 2^-22). A second rounding to 16 bits
    anywhere would give 1.4 times as much."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, T + E + D)
    gu, gv = _stack(cuda, g, E, 2 * I, D, D ** -0.5)
    dn, dv = _stack(cuda, g, E, D, I, I ** -0.5)
    x = torch.randn((T, D), generator=g, device=cuda).to(_dt(dtype))
    inds = torch.rand((T, E), generator=g, device=cuda).topk(k, -1).indices.to(torch.int32)
    weights = 0.5 + torch.rand((T, k), generator=g, device=cuda)
    want = _experts(x, inds, weights, gv, dv)
    y = fp4.experts(x, inds, weights, gu, dn)
    assert _status(cuda) == 0
    off, once = _rms(y.double() - want), _rms(want.to(_dt(dtype)).double() - want)
    assert off <= 1.05 * once
    assert torch.equal(y, fp4.experts(x, inds, weights, gu, dn))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,k,D,I", [(1, 2, 130, 64), (20, 3, 130, 64), (300, 2, 101, 37), (20, 2, 128, 33)])
def test_switch_glu_takes_any_width(cuda, dtype, T, k, D, I):
    """Each slot's output is rounded once and its hidden row once before it; the two add in squares. A rounding's error relative to
    the value is twice as large at the lower end of a power of two as at the upper, and few hidden values make most of an output
    (33 of them, of a long-tailed distribution), so the hidden rows' may be up to twice the output's: 5 ** 0.5 = 2.24 of it."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, T + D)
    E = 4
    gu, gv = _stack(cuda, g, E, 2 * I, D, D ** -0.5)
    dn, dv = _stack(cuda, g, E, D, I, I ** -0.5)
    x = torch.randn((T, D), generator=g, device=cuda).to(_dt(dtype))
    inds = torch.rand((T, E), generator=g, device=cuda).topk(k, -1).indices.to(torch.int32)
    ys = fp4.switch_glu(x, inds, gu, dn)
    assert _status(cuda) == 0 and ys.shape == (T, k, D)
    one = torch.ones((T, 1), device=cuda)
    want = torch.stack([_experts(x, inds[:, r:r + 1], one, gv, dv) for r in range(k)], 1)
    off, once = _rms(ys.double() - want), _rms(want.to(_dt(dtype)).double() - want)
    assert off <= 2.3 * once


def _poison(cuda):
    """Memory that the allocator hands out next holds no numbers."""
    import torch

    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24):
        t = torch.full((n,), float("nan"), device=cuda)
        del t


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,k,D", [(1, 4, 256), (1, 3, 101), (20, 2, 256), (20, 3, 130), (300, 2, 256), (1200, 2, 128)])
def test_experts_leave_ids_out_that_are_no_experts(cuda, dtype, T, k, D):
    """Ids of -1 and beyond the last expert add nothing, and are recorded; a token of none but those is zeros."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, T + k)
    E, I = 5, 96
    gu, gv = _stack(cuda, g, E, 2 * I, D, D ** -0.5)
    dn, dv = _stack(cuda, g, E, D, I, I ** -0.5)
    x = torch.randn((T, D), generator=g, device=cuda).to(_dt(dtype))
    weights = 0.5 + torch.rand((T, k), generator=g, device=cuda)
    for bad in (-1, E, 1 << 30, -2 ** 31):
        inds = torch.randint(0, E, (T, k), generator=g, device=cuda).to(torch.int32)
        inds[::2, 0] = bad
        if T > 1:
            inds[1] = bad
        _poison(cuda)
        y = fp4.experts(x, inds, weights, gu, dn)
        assert _status(cuda) == 2  # LQ_DEV_BOUNDS
        want = _experts(x, inds, weights, gv, dv)
        assert bool(torch.isfinite(y).all()) and (T == 1 or not bool(y[1].any()))
        off, once = _rms(y.double() - want), _rms(want.to(_dt(dtype)).double() - want)
        assert off <= 1.05 * once
        if T > 1:
            ys = fp4.switch_glu(x, inds, gu, dn)
            assert _status(cuda) == 2
            assert not bool(ys[(inds < 0) | (inds >= E)].any()) and bool(torch.isfinite(ys).all())


@pytest.mark.parametrize("T,k,E", [(1, 2, 4), (40, 3, 6), (200, 2, 40), (1500, 2, 6)])
def test_a_grouping_marks_pairs_of_no_expert_and_its_readers_skip_them(cuda, T, k, E):
    import torch
    from locals_b200 import moe

    g = _gen(cuda, T)
    inds = torch.randint(-1, E + 1, (T, k), generator=g, device=cuda).to(torch.int32)
    inds[0, 0] = -1
    _poison(cuda)
    order, starts, experts, nseg, pos = moe.group(inds, E)
    assert _status(cuda) == 2
    flat = inds.reshape(-1)
    fine = (flat >= 0) & (flat < E)
    n = int(fine.sum())
    want = torch.argsort(torch.where(fine, flat, E), stable=True)[:n]
    assert torch.equal(order[:n].long(), want) and bool((order[n:] == -1).all())
    assert bool((pos[~fine] == -1).all()) and torch.equal(pos[want].long(), torch.arange(n, device=cuda))
    assert int(starts[int(nseg)]) == n
    x = torch.randn((T, 64), generator=g, device=cuda).to(torch.bfloat16)
    xs = moe.gather(x, order, k)
    assert torch.equal(xs[:n], x[want // k]) and not bool(xs[n:].any())
    ys = torch.randn((T * k, 64), generator=g, device=cuda).to(torch.bfloat16)
    w = torch.rand((T, k), generator=g, device=cuda)
    kept = torch.where(fine[:, None], ys[pos.long().clamp(min=0)], torch.zeros_like(ys))  # the same sums, of zeros in their place
    a, b = moe.combine(ys, w, pos), moe.combine(kept, w, None)
    assert torch.equal(a, b)
    odd = moe.combine(ys[:, :63].contiguous(), w, pos)  # one column a thread
    assert torch.equal(odd, b[:, :63])
    res, nw = torch.randn((T, 64), generator=g, device=cuda).to(torch.bfloat16), torch.ones(64, device=cuda, dtype=torch.bfloat16)
    for p, q in zip(moe.combine_norm(ys, w, pos, res, nw, 1e-5), moe.combine_norm(kept, w, None, res, nw, 1e-5)):
        assert torch.equal(p, q)
    assert _status(cuda) == 0


def test_one_tokens_affine_down_projection_skips_a_pair_of_no_expert(cuda):
    import torch
    from locals_b200 import moe

    g = _gen(cuda, 4)
    E, D, I = 4, 256, 512
    w = torch.randint(-2 ** 31, 2 ** 31, (E, D, I // 8), generator=g, device=cuda).to(torch.int32)
    s, b = (torch.rand((E, D, I // 64), generator=g, device=cuda).to(torch.bfloat16) * 0.01 for _ in range(2))
    h = torch.randn((3, I), generator=g, device=cuda).to(torch.bfloat16)
    weights = torch.rand((1, 3), generator=g, device=cuda)
    grouping = moe.group(torch.tensor([[2, -1, 0]], device=cuda, dtype=torch.int32), E)
    assert _status(cuda) == 2
    y = moe.down_combine(h, grouping, weights, (w, s, b))
    assert y is not None and _status(cuda) == 2
    rest = moe.group(torch.tensor([[2, 0]], device=cuda, dtype=torch.int32), E)
    want = moe.down_combine(h[:2].contiguous(), rest, weights[:, [0, 2]].contiguous(), (w, s, b))
    assert torch.equal(y, want)


@pytest.mark.parametrize("P,gather", [(4, 2), (4, 3), (200, 2), (700, 5)])
def test_a_negative_row_to_gather_is_recorded_and_zeros(cuda, P, gather):
    """-1 .. -(gather - 1) are no rows either (divided, they would be row 0): in the product that makes its pieces itself (few rows)
    and in the split before it."""
    import torch
    from locals_b200 import _lib
    from locals_b200.kernels import _stream

    g = _gen(cuda, P)
    N, K = 64, 128
    w, wv = _stack(cuda, g, 1, N, K)
    x = torch.randn((P, K), generator=g, device=cuda).to(torch.bfloat16)
    order = torch.arange(P, device=cuda, dtype=torch.int32) * gather
    bad = torch.tensor([1, P // 2, P - 1], device=cuda)
    order[bad] = torch.tensor([-1, 1 - gather, -2 ** 31], device=cuda, dtype=torch.int32)
    starts, ids, nseg = (torch.tensor(v, device=cuda, dtype=torch.int32) for v in ([0, P], [0], [1]))
    out = torch.full((P, N), 5.0, device=cuda, dtype=torch.bfloat16)
    n = _lib.lib().lq_fp4_experts_workspace(P, P, 1, N, K, _lib.BF16)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    _lib.call("lq_fp4_experts", x.data_ptr(), P, order.data_ptr(), gather, starts.data_ptr(), ids.data_ptr(), nseg.data_ptr(), P, P, 0,
              w.codes.data_ptr(), w.tiles.data_ptr(), out.data_ptr(), 1, N, K, _lib.BF16, ws.data_ptr() if n else None, n, _stream())
    assert _status(cuda) == 2
    assert not bool(out[bad].any())
    keep = torch.ones(P, dtype=torch.bool, device=cuda)
    keep[bad] = False
    want, bound = R.linear(x[keep], wv[0], torch.bfloat16)
    assert bool(((out[keep].double() - want).abs() <= bound).all())


# ---- quantize, and the matrices' factors -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,K", [(1, 16), (3, 40), (200, 640)])
def test_a_matrix_of_zeros_with_its_own_factor_is_zeros(cuda, dtype, rows, K):
    """Its largest magnitude / 2688 is 0: scales and codes are 0, and so is every product with it."""
    import torch
    from locals_b200 import fp4

    x = torch.zeros((rows, K), device=cuda, dtype=_dt(dtype))
    x[:, ::3] = -0.0
    f = (x.float().abs().amax() / 2688).reshape(1)
    assert float(f) == 0
    _poison(cuda)
    a = fp4.quantize(x, "nvfp4", scale=f)
    assert not bool(a.codes.any()) and not bool(fp4.unpack(a)[1].any())
    assert bool((fp4.dequantize(a, torch.float32) == 0).all())
    w = torch.randn((70, K), generator=_gen(cuda, K), device=cuda)
    fw = (w.abs().amax() / 2688).reshape(1)
    q = fp4.quantize(w, "nvfp4", scale=fw)
    for y in (fp4.matmul(a, q, dtype=torch.float32), fp4.matmul(q, a, dtype=torch.float32), fp4.matmul(a, q, dtype=torch.float32, glu=True)):
        assert bool((y == 0).all())
    assert _status(cuda) == 0


@pytest.mark.parametrize("M,N,K", [(1, 96, 256), (17, 130, 64), (70, 96, 256), (300, 257, 256)])
@pytest.mark.parametrize("fx,fw", [(1e-22, 3e-22), (1e-30, 1e-10), (2e25, 1e25), (1e-40, 1e30), (3e38, 3e38), (1e-45, 1e-45), (0.7, 1.3)])
def test_factors_near_the_ends_of_the_range(cuda, M, N, K, fx, fw):
    """A product of factors that 32 bits do not hold does not spoil sums that its result does: 0 stays 0, and what is a normal
    number has its bits."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M)

    def operand(rows, f, zero):
        codes = torch.randint(0, 16, (rows, K), generator=g, device=cuda, dtype=torch.int32)
        byte = torch.randint(1, 127, (rows, K // 16), generator=g, device=cuda).to(torch.uint8)
        codes[zero] = 0
        words = (codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=cuda, dtype=torch.int32))).sum(-1, dtype=torch.int32)
        t = torch.tensor([f], device=cuda)
        return fp4.pack(words, byte, "nvfp4", t), R.values(codes, byte, "nvfp4", K), t.double()

    x, xv, dx = operand(M, fx, 0)
    w, wv, dw = operand(N, fw, 1)
    f = dx * dw
    want = (xv @ wv.T) * f
    y = fp4.matmul(x, w, dtype=torch.float32)
    assert _status(cuda) == 0
    assert bool((y[0] == 0).all()) and bool((y[:, 1] == 0).all())
    top = torch.finfo(torch.float32).max
    # sums in 32 bits; the product of the factors, and its product with a sum, rounded once each; what is no normal number to the step there
    bound = R.lost(K, xv, wv) * f + 2.0 ** -22 * want.abs() + 2 * 2.0 ** -149
    fine = want.abs() + bound < top
    assert bool(((y.double() - want).abs() <= bound)[fine].all())
    over = want.abs() - bound > top * (1 + 2.0 ** -24)
    assert torch.equal(y[over], (torch.sign(want) * float("inf")).float()[over])


# ---- SwiGLU ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M", [1, 20, 70, 200, 300])
def test_glu_of_gates_far_below_zero(cuda, mode, M):
    """silu in 32 bits has its bits where the gate is -10 to -100. expf is off by one unit in the last place (2^-23 of the value at
    most), the fast quotient by two for divisors in range, the sum with 1, the product and the product with up round once each
    (2^-24): 3 * 2^-23 + 3 * 2^-24 in all; where e^gate is no normal number, that is off by a step of 2^-149 at most, which the gate
    and up (64) multiply."""
    import torch
    from locals_b200 import fp4

    K, gates = 32, [-0.5 * i for i in range(0, 201)] + [0.5 * i for i in range(1, 41)]
    left = torch.tensor(gates).double()
    codes = torch.zeros((len(gates), 2, K), dtype=torch.int32)
    values = [6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5]
    for k in range(K):  # each gate as a sum of K values, the largest first
        for c, v in zip(range(7, 0, -1), values):
            take = (left.abs() >= v) & (codes[:, 0, k] == 0)
            codes[take, 0, k] = torch.where(left[take] < 0, c + 8, c).to(torch.int32)
            left = torch.where(take, left - torch.sign(left) * v, left)
    assert not left.any()
    codes[:, 1, :16] = 6  # up: 16 times 4
    words = (codes.flatten(0, 1).unflatten(-1, (-1, 8)) << (4 * torch.arange(8, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    one = 127 if mode == "mxfp4" else 0x38
    w = fp4.pack(words.to(cuda), torch.full((2 * len(gates), K // R.GROUP[mode]), one, dtype=torch.uint8, device=cuda), mode)
    x = fp4.pack(torch.full((M, K // 8), 0x22222222, dtype=torch.int32, device=cuda),
                 torch.full((M, K // R.GROUP[mode]), one, dtype=torch.uint8, device=cuda), mode)
    y = fp4.matmul(x, w, dtype=torch.float32, glu=True)
    assert _status(cuda) == 0
    g = torch.tensor(gates, dtype=torch.float64, device=cuda)
    want = 64 * g / (1 + torch.exp(-g))
    bound = (3 * 2.0 ** -23 + 3 * 2.0 ** -24) * want.abs() + 2.0 ** -149 * 64 * g.abs() + 2.0 ** -149
    assert bool(((y.double() - want).abs() <= bound).all())


# ---- dequantize ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("f", [1e-38, 3e-40, 1.0, 1e35, 3e38])
def test_dequantize_with_factors_near_the_ends_of_the_range(cuda, dtype, f):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 7)
    codes = torch.randint(0, 16, (40, 96), generator=g, device=cuda, dtype=torch.int32)
    byte = torch.randint(0, 127, (40, 6), generator=g, device=cuda).to(torch.uint8)
    words = (codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=cuda, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    scale = torch.tensor([f], device=cuda)
    want = R.values(codes, byte, "nvfp4", 96, scale)
    got = fp4.dequantize(fp4.pack(words, byte, "nvfp4", scale), _dt(dtype)).double()
    i = torch.finfo(_dt(dtype))
    over = want.abs() >= i.max * (1 + R.half_step(_dt(dtype))) * (1 + 2.0 ** -23)
    assert torch.equal(got[over], torch.sign(want[over]) * float("inf"))
    # half a step of the type, and half a step of 32 bits for the product with the factor before it
    once = torch.maximum(R.half_step(_dt(dtype)) * want.abs(), torch.tensor(i.smallest_normal * i.eps / 2, dtype=torch.float64, device=cuda))
    bound = once + torch.maximum(2.0 ** -24 * want.abs(), torch.tensor(2.0 ** -150, dtype=torch.float64, device=cuda))
    under = want.abs() <= i.max
    assert bool(((got - want).abs() <= bound)[under].all())


# ---- 16 bits by 4, long rows -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M", [1, 20, 70, 300])
@pytest.mark.parametrize("K", [4096, 9728, 14336])
def test_linear_picks_single_values_out_of_long_rows(cuda, dtype, M, K):
    """Each row of w picks one value of x by a code of 1 and a scale of 1: all of its bits, from every piece, wherever it stands."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, M + K)
    N = 512
    at = torch.randperm(K, generator=g, device=cuda)[:N]
    at[:4] = torch.tensor([0, 31, K - 32, K - 1], device=cuda)
    words = torch.zeros((N, K // 8), dtype=torch.int32, device=cuda)
    words[torch.arange(N, device=cuda), at // 8] = (2 << (4 * (at % 8))).to(torch.int32)
    w = fp4.pack(words, torch.full((N, K // 32), 127, dtype=torch.uint8, device=cuda))
    x = (1 + torch.rand((M, K), generator=g, device=cuda)) * torch.exp2(torch.randint(-12, 1, (M, K), generator=g, device=cuda).float())
    x = torch.where(torch.rand((M, K), generator=g, device=cuda) < 0.5, -x, x).to(_dt(dtype))
    assert torch.equal(fp4.matmul(x, w), x[:, at])
    assert _status(cuda) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 2048, 9728), (20, 512, 9728), (70, 512, 9728), (300, 512, 14336), (2, 4096, 4096)])
def test_linear_over_long_rows_is_rounded_once(cuda, dtype, M, N, K):
    """Sums in 32 bits add little to one rounding of the result: 1,344 steps (K / 32 of three pieces) of 2^-22 of a sum are 2^-17 of it in
    their mean square, a twentieth of a rounding to fp16 (2^-12.8), so 1.002 in squares. Without its last piece a value is off by up to
    2^-4 (bf16) or 2^-9 (fp16), several roundings."""
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, N + K)
    w = fp4.quantize(torch.randn((N, K), generator=g, device=cuda) * 0.02)
    x = torch.randn((M, K), generator=g, device=cuda).to(_dt(dtype))
    want = x.double() @ fp4.dequantize(w, torch.float32).double().T
    off, once = _rms(fp4.matmul(x, w).double() - want), _rms(want.to(_dt(dtype)).double() - want)
    assert _status(cuda) == 0
    assert off <= 1.05 * once


@pytest.mark.parametrize("T,k,E,D,I", [(34, 2, 4, 256, 96), (17, 1, 1, 128, 64), (2, 17, 2, 128, 64), (1, 5, 8, 128, 64), (300, 4, 8, 130, 66)])
def test_routed_experts_stay_within_their_workspace(cuda, T, k, E, D, I):
    import torch
    from locals_b200 import _lib
    from locals_b200.kernels import _stream

    g = _gen(cuda, T)
    gu, gv = _stack(cuda, g, E, 2 * I, D, D ** -0.5)
    dn, dv = _stack(cuda, g, E, D, I, I ** -0.5)
    x = torch.randn((T, D), generator=g, device=cuda).to(torch.bfloat16)
    inds = torch.randint(0, E, (T, k), generator=g, device=cuda).to(torch.int32)
    weights = 0.5 + torch.rand((T, k), generator=g, device=cuda)
    n = _lib.lib().lq_fp4_moe_workspace(T, k, E, D, I, _lib.BF16)
    ws = torch.full((n + (1 << 22),), 0xA5, dtype=torch.uint8, device=cuda)
    y = torch.full((T + 4, D), 7.0, dtype=torch.bfloat16, device=cuda)
    _lib.call("lq_fp4_moe", x.data_ptr(), inds.data_ptr(), weights.data_ptr(), gu.codes.data_ptr(), gu.tiles.data_ptr(), dn.codes.data_ptr(),
              dn.tiles.data_ptr(), y.data_ptr(), T, k, E, D, I, _lib.BF16, ws.data_ptr(), n, _stream())
    assert _status(cuda) == 0
    assert bool((ws[n:] == 0xA5).all()) and bool((y[T:] == 7.0).all())
    want = _experts(x, inds, weights, gv, dv)
    off, once = _rms(y[:T].double() - want), _rms(want.to(torch.bfloat16).double() - want)
    assert off <= 1.05 * once


def test_more_experts_than_segments_are_refused(cuda):
    import torch
    from locals_b200 import fp4

    E, D, I = 1025, 32, 32
    gu = fp4.Fp4(torch.zeros((E, 2 * I, 16), dtype=torch.int32, device=cuda), torch.full((E, 1, 1, 512), 127, dtype=torch.uint8, device=cuda), "mxfp4", D)
    dn = fp4.Fp4(torch.zeros((E, D, 16), dtype=torch.int32, device=cuda), torch.full((E, 1, 1, 512), 127, dtype=torch.uint8, device=cuda), "mxfp4", I)
    x = torch.ones((600, D), dtype=torch.bfloat16, device=cuda)
    for T, k in ((600, 2), (1, 1025)):
        inds, weights = torch.zeros((T, k), dtype=torch.int32, device=cuda), torch.ones((T, k), device=cuda)
        with pytest.raises(Exception, match="shape"):
            fp4.experts(x[:T], inds, weights, gu, dn)
    few = torch.full((300, 2), 1024, dtype=torch.int32, device=cuda)  # 600 pairs of the same stack are answered
    assert not bool(fp4.experts(x[:300], few, torch.ones((300, 2), device=cuda), gu, dn).any())
    assert _status(cuda) == 0


# ---- refusals ------------------------------------------------------------------------------------------------

def test_glu_of_an_odd_number_of_rows_is_refused(cuda):
    import torch
    from locals_b200 import fp4

    g = _gen(cuda, 1)
    w = fp4.quantize(torch.randn((95, 128), generator=g, device=cuda))
    x = torch.randn((4, 128), generator=g, device=cuda).to(torch.bfloat16)
    for a in (x, fp4.quantize(x)):
        assert fp4.matmul(a, w).shape == (4, 95)
        with pytest.raises(ValueError, match="gate and up"):
            fp4.matmul(a, w, glu=True)
    assert _status(cuda) == 0


def test_pairs_without_tokens_are_refused(cuda):
    """They were answered with whatever the memory held."""
    import torch
    from locals_b200 import fp4, moe

    g = _gen(cuda, 1)
    w, _ = _stack(cuda, g, 3, 64, 128)
    grouping = moe.group(torch.tensor([0, 2, 1, 1], device=cuda, dtype=torch.int32), 3)
    x = torch.randn((2, 128), generator=g, device=cuda).to(torch.bfloat16)
    assert fp4.grouped(x, grouping, w, 2, gather_k=2).shape == (4, 64)
    with pytest.raises(ValueError):
        fp4.grouped(x[:0], grouping, w, 2, gather_k=2)
    with pytest.raises(ValueError):
        fp4.grouped(x, grouping, w, 0, gather_k=2)
    none = tuple(torch.empty(n, device=cuda, dtype=torch.int32) for n in (0, 1, 0, 1, 0))
    assert fp4.grouped(x[:0], none, w, 1, gather_k=2).shape == (0, 64)
    assert _status(cuda) == 0


@pytest.mark.parametrize("P", [8, 96, 800])
def test_a_grouping_of_more_experts_than_the_stack_has_is_recorded(cuda, P):
    """Segments of experts that the stack does not have are left out; those that it has are answered."""
    import torch
    from locals_b200 import fp4, moe

    g = _gen(cuda, P)
    w, wv = _stack(cuda, g, 3, 64, 128)
    inds = torch.arange(P, device=cuda, dtype=torch.int32) % 8
    grouping = moe.group(inds, 8)
    x = torch.randn((P, 128), generator=g, device=cuda).to(torch.bfloat16)
    got = fp4.grouped(x, grouping, w, P)
    assert _status(cuda) == 2  # LQ_DEV_BOUNDS
    ids = inds[grouping[0].long()]
    for e in range(3):
        want, bound = R.linear(x[ids == e], wv[e], torch.bfloat16)
        assert bool(((got[ids == e].double() - want).abs() <= bound).all())


# ---- host threads ----------------------------------------------------------------------------------------------

def _at_once(calls, rounds=3000):
    """Each call over and over on a host thread and stream of its own (the C ABI's calls run without the interpreter's lock): their
    return codes."""
    import threading

    import torch

    codes, go = [set() for _ in calls], threading.Barrier(len(calls))

    def work(i, call, stream):
        torch.cuda.set_device(0)
        go.wait()
        for _ in range(rounds):
            codes[i].add(call(stream))

    streams = [torch.cuda.Stream() for _ in calls]
    threads = [threading.Thread(target=work, args=(i, c, s.cuda_stream)) for i, (c, s) in enumerate(zip(calls, streams))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return codes


def test_dense_and_grouped_products_of_two_host_threads(cuda):
    """They run the same kernel with shared memory of different sizes."""
    import torch
    from locals_b200 import _lib

    L, g = _lib.lib(), _gen(cuda, 3)
    N, K, M, P = 128, 256, 40, 96
    w, wv = _stack(cuda, g, 2, N, K)
    x = torch.randn((P, K), generator=g, device=cuda).to(torch.bfloat16)
    starts, ids, nseg = (torch.tensor(v, device=cuda, dtype=torch.int32) for v in ([0, 50, P], [0, 1], [2]))
    y, z = (torch.zeros((n, N), device=cuda, dtype=torch.bfloat16) for n in (M, P))
    n1, n2 = L.lq_fp4_linear_workspace(M, N, K, _lib.BF16), L.lq_fp4_experts_workspace(P, P, 2, N, K, _lib.BF16)
    w1, w2 = (torch.empty(max(n, 1), device=cuda, dtype=torch.uint8) for n in (n1, n2))
    torch.cuda.synchronize()

    def dense(st):
        return L.lq_fp4_linear(x.data_ptr(), K, w.codes.data_ptr(), w.tiles.data_ptr(), M, N, K, 0, _lib.BF16, y.data_ptr(), w1.data_ptr(), n1, st)

    def grouped(st):
        return L.lq_fp4_experts(x.data_ptr(), P, None, 0, starts.data_ptr(), ids.data_ptr(), nseg.data_ptr(), P, P, 0, w.codes.data_ptr(),
                                w.tiles.data_ptr(), z.data_ptr(), 2, N, K, _lib.BF16, w2.data_ptr(), n2, st)

    assert _at_once([dense, grouped]) == [{0}, {0}]
    assert _status(cuda) == 0
    for got, rows, m in ((y, slice(0, M), wv[0]), (z[:50], slice(0, 50), wv[0]), (z[50:], slice(50, P), wv[1])):
        want, bound = R.linear(x[rows], m, torch.bfloat16)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_groupings_of_two_host_threads(cuda):
    import torch
    from locals_b200 import _lib

    L, P, calls, keep = _lib.lib(), 2500, [], []
    for E in (400, 1024):
        ids = (torch.arange(P, device=cuda, dtype=torch.int32) * 7) % E
        b = [torch.empty(n, device=cuda, dtype=torch.int32) for n in (P, E + 1, E, 1, P)]
        keep.append((ids, b, E))
        calls.append(lambda st, a=(ids.data_ptr(), P, E, *(t.data_ptr() for t in b)): L.lq_moe_group(*a, st))
    torch.cuda.synchronize()
    assert _at_once(calls) == [{0}, {0}]
    assert _status(cuda) == 0
    for ids, b, E in keep:
        assert torch.equal(b[0].long(), torch.argsort(ids, stable=True))
