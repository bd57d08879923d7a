"""Activations in 8 bits: the packed form bit by bit, what is computed from it against 64 bits.

Tolerances: a GELU or its derivative is off by the error of a 32-bit erf and exp (8 x 2^-24 of the terms' size) and half a step of
the output's type; a weight gradient sums M exact products in 32 bits: M 2^-24 sum |dy x| whatever the order."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TD = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    import sitk  # noqa: F401
    from sitk import ops as _ops
    return _ops


def steps_ref(x):
    """(codes, exponents) of the rows by the definition: the smallest step whose largest code is at most 127."""
    rows, cols = x.shape
    xd = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, -1, 32)
    amax = xd.abs().amax(-1, keepdim=True)
    k = torch.full_like(amax, -24.0 if x.dtype == torch.float16 else -126.0)
    k = torch.maximum(k, torch.floor(torch.log2(amax.clamp_min(1e-300))) - 8)
    for _ in range(4):
        k = torch.where((amax * torch.exp2(-k)).round() > 127, k + 1, k)
    k = k.clamp_max(9 if x.dtype == torch.float16 else 121)   # a larger step could read back as infinity: codes end at 127 there
    return (xd * torch.exp2(-k)).round().clamp(-127, 127), k


def value_ref(x):
    q, k = steps_ref(x)
    return (q * torch.exp2(k)).view(x.shape[0], -1)[:, :x.shape[1]]


def sample(rows, cols, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows * 7 + cols)
    return (torch.randn(rows, cols, device=DEV, generator=g) * torch.exp(torch.randn(1, cols, device=DEV, generator=g))).to(TD[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (321, 192), (77, 612), (2, 4097), (1000, 64)])
def test_pack_is_exact(ops, dtype, rows, cols):
    x = sample(rows, cols, dtype)
    p = ops.act8_pack(x)
    q, k = steps_ref(x)
    assert torch.equal(p.codes.view(rows, -1, 32).double(), q)
    assert torch.equal(p.steps.double() - 127, k[..., 0])
    y = ops.act8_unpack(p)
    assert y.dtype == x.dtype and y.shape == x.shape and torch.equal(y.double(), value_ref(x))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_pack_at_the_borders(ops, dtype):
    """The largest and smallest values of the type, zeros, ties between codes, the largest code's own tie (127.5)."""
    t = TD[dtype]
    fi = torch.finfo(t)
    rows = [[fi.max, -fi.max], [fi.tiny, -fi.tiny], [fi.smallest_normal / 8, 0.0], [0.0, -0.0], [127.5, 1.5], [127.0, 2.5], [1.9921875, 0.5 / 64],
            [255.0, 3.0], [2.0 ** -24, 2.0 ** -23], [64.0, 0.25], [1.0, 1.0 / 128]]
    x = torch.zeros(len(rows), 32, device=DEV, dtype=t)
    x[:, 5:7] = torch.tensor(rows, device=DEV, dtype=torch.float64).to(t)
    y = ops.act8_unpack(ops.act8_pack(x))
    assert torch.equal(y.double(), value_ref(x))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_non_finite_values_stay_in_their_group(ops, dtype):
    x = sample(4, 96, dtype)
    x[0, 3], x[1, 40], x[2, 95] = math.nan, math.inf, -math.inf
    y = ops.act8_unpack(ops.act8_pack(x))
    bad = torch.zeros(4, 3, dtype=torch.bool, device=DEV)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(torch.isnan(y).view(4, 3, 32), bad[..., None].expand(4, 3, 32))


def test_pack_strides(ops):
    x = sample(40, 200, "bf16")
    for v in (x[:, :64], x[:, 3:70], x[::3], x.t(), x[:1].expand(9, 200), x.view(4, 10, 200), x[:, 0]):
        y = ops.act8_unpack(ops.act8_pack(v))
        assert y.shape == v.shape
        assert torch.equal(y.double().reshape(-1, v.shape[-1]), value_ref(v.reshape(-1, v.shape[-1]).contiguous()))
    e = ops.act8_pack(torch.empty(0, 17, device=DEV))
    assert ops.act8_unpack(e).shape == (0, 17)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 33), (321, 768), (50, 612)])
def test_gelu_and_its_gradient(ops, dtype, rows, cols):
    u = 2 * sample(rows, cols, dtype)
    if u.numel() > 16:
        u.view(-1)[:6] = torch.tensor([0.0, -0.0, 30.0, -30.0, 5.5, -5.5], device=DEV, dtype=u.dtype)
    dg = sample(rows, cols, dtype, seed=5)
    eps = torch.finfo(TD[dtype]).eps / 2
    tiny = torch.finfo(TD[dtype]).smallest_normal
    g, p = ops.act8_gelu_fwd(u)
    ud = u.double()
    want = 0.5 * ud * torch.special.erfc(-ud / math.sqrt(2))
    # 1 + erf loses 2^-24 of its terms
    assert bool(((g.double() - want).abs() <= eps * want.abs() + 8 * 2.0 ** -24 * ud.abs() + tiny).all())
    assert torch.equal(ops.act8_unpack(p).double(), value_ref(u))
    du = ops.act8_gelu_bwd(dg, p)
    u8 = value_ref(u)
    d = 0.5 * torch.special.erfc(-u8 / math.sqrt(2)) + u8 * torch.exp(-0.5 * u8 * u8) / math.sqrt(2 * math.pi)
    want = dg.double() * d
    assert bool(((du.double() - want).abs() <= eps * want.abs() + 16 * 2.0 ** -24 * dg.double().abs() + tiny).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (2, 1, 1), (33, 40, 45), (64, 64, 64), (321, 192, 612), (1000, 136, 100), (4100, 72, 260),
                                   (20001, 64, 96)])
def test_wgrad(ops, dtype, M, N, K):
    x, dy = sample(M, K, dtype), sample(M, N, dtype, seed=9)
    p = ops.act8_pack(x)
    x8 = value_ref(x)
    dW, db = ops.act8_wgrad(dy, p)
    tol = (M + 8) * 2.0 ** -24
    want, mag = dy.double().t() @ x8, dy.double().abs().t() @ x8.abs()
    assert bool(((dW.double() - want).abs() <= tol * mag + 2.0 ** -24 * want.abs()).all())
    assert bool(((db.double() - dy.double().sum(0)).abs() <= tol * dy.double().abs().sum(0)).all())
    again = ops.act8_wgrad(dy, p)
    assert torch.equal(again[0], dW) and torch.equal(again[1], db)
    # added to what is there, inside a wider buffer
    buf = torch.full((N, K + 3), 2.0, device=DEV)
    b2 = torch.full((N,), 3.0, device=DEV)
    ops.act8_wgrad(dy, p, dW=buf[:, :K], db=b2)
    assert bool(((buf[:, :K].double() - 2 - want).abs() <= tol * mag + 2.0 ** -23 * (2 + want.abs())).all())
    assert bool((buf[:, K:] == 2).all())
    assert bool(((b2.double() - 3 - dy.double().sum(0)).abs() <= tol * dy.double().abs().sum(0) + 2.0 ** -23 * (3 + db.double().abs())).all())
    buf.fill_(1.0)
    ops.act8_wgrad(dy, p, dW=buf[:, :K])
    assert bool(((buf[:, :K].double() - 1 - want).abs() <= tol * mag + 2.0 ** -23 * (1 + want.abs())).all())


def test_wgrad_strides_and_no_rows(ops):
    x = sample(100, 64, "bf16")
    p = ops.act8_pack(x)
    wide = sample(100, 70, "bf16", seed=3)
    want, mag = wide[:, :24].double().t() @ value_ref(x), wide[:, :24].double().abs().t() @ value_ref(x).abs()
    for d in (wide[:, :24].contiguous(), wide[:, :24], wide[:, 1:25].clone(), torch.cat([wide, wide], 1)[:, 70:94]):
        got = ops.act8_wgrad(d, p)                    # rows of 16-byte steps and others: two kernels, sums in their own order
        w, g = (want, mag) if torch.equal(d, wide[:, :24]) else (d.double().t() @ value_ref(x), d.double().abs().t() @ value_ref(x).abs())
        assert bool(((got[0].double() - w).abs() <= 108 * 2.0 ** -24 * g + 2.0 ** -24 * w.abs()).all())
    e = ops.act8_wgrad(wide[:1, :24].expand(100, 24), p)
    want = wide[:1, :24].double().expand(100, 24).t() @ value_ref(x)
    assert float((e[0].double() - want).abs().max()) <= 108 * 2.0 ** -24 * float((wide[:1, :24].double().abs().t() * value_ref(x).abs().sum(0)).max())
    dW, db = ops.act8_wgrad(torch.empty(0, 24, device=DEV), ops.act8_pack(torch.empty(0, 40, device=DEV)))
    assert dW.shape == (24, 40) and float(dW.abs().max()) == 0.0 and float(db.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N", [24, 21])
def test_wgrad_without_rows(ops, dtype, N):
    """Zeros in every element, rows of a wider buffer left as they are; added to a gradient: that gradient, bit for bit."""
    p = ops.act8_pack(torch.empty(0, 40, device=DEV, dtype=TD[dtype]))
    dy = torch.empty(0, N, device=DEV, dtype=TD[dtype])
    junk = [torch.full((N, 40), math.nan, device=DEV) for _ in range(8)]       # what the allocator hands out next
    del junk
    dW, db = ops.act8_wgrad(dy, p)
    assert dW.shape == (N, 40) and not dW.any() and db.shape == (N,) and not db.any()
    wide = torch.randn(N, 43, device=DEV)
    was, b = wide.clone(), torch.randn(N, device=DEV)
    b_was = b.clone()
    ops.act8_wgrad(dy, p, dW=wide[:, 1:41], db=b)
    assert torch.equal(wide, was) and torch.equal(b, b_was)
