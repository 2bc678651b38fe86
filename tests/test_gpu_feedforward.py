"""Feed-forward, 8-bit and distillation operators of ``ops`` on the MI355X.

Every output is compared element by element with the definition in 64 bits.
The bounds are worst cases of the arithmetic that the kernels document:

  * a sum of K products in 32 bits: each of the K additions is off by at most
    2^-23 of the partial sum (a matrix unit may truncate), so by at most
    K 2^-23 sum_k |a_k b_k| in all;
  * a rounding to bf16 is off by at most 2^-8 of the value, to fp32 2^-24;
  * an activation in 32 bits by a few units in the last place (2^-20 allowed).
"""

import ctypes
import math

import pytest
import torch

import mpi_cuda_cnn_amd.ops as ops

D64 = torch.float64
EPS_SUM = 2.0**-23
EPS_BF16 = 2.0**-8
EPS_F32 = 2.0**-24
EPS_ACT = 2.0**-20


def gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device=g.device, generator=g) * std).to(dtype)


def within(got, ref, bound, what=""):
    """|got - ref| <= bound everywhere; NaN and infinities at the same places."""
    got = got.to(D64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got)), what
    over = ((got - ref).abs() - bound)[fin]
    assert over.numel() == 0 or over.max().item() <= 0, (what, over.max().item(), int((over > 0).sum()))


def act64(v, act):
    """(f, f') in 64 bits."""
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * c, c + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        return v.clamp(min=0), (v > 0).to(v.dtype)
    if act == "tanh":
        t = torch.tanh(v)
        return t, 1 - t * t
    return v, torch.ones_like(v)


# ---------------------------------------------------------------------------------------------------------------
# gated_linear
# ---------------------------------------------------------------------------------------------------------------
def gated_check(x, wg, wu, act, out, save):
    X, G, U = x.to(D64), wg.to(D64), wu.to(D64)
    K = x.shape[1]
    g, u = X @ G.t(), X @ U.t()
    dg = K * EPS_SUM * (X.abs() @ G.abs().t())
    du = K * EPS_SUM * (X.abs() @ U.abs().t())
    f, _ = act64(g, act)
    # |f'| <= 1.13 for all of them
    df = 1.13 * dg + EPS_ACT * (f.abs() + g.abs() * 2.0**-3)
    ref = f * u
    err = df * u.abs() + (f.abs() + df) * du + EPS_F32 * ref.abs()
    h = out[0] if save else out
    within(h, ref, err + EPS_BF16 * (ref.abs() + err) + 1e-38, "h")
    if save:
        within(out[1], g, dg + EPS_BF16 * (g.abs() + dg) + 1e-38, "gate")
        within(out[2], u, du + EPS_BF16 * (u.abs() + du) + 1e-38, "up")


GATED = [(1, 64, 16), (1, 8, 1), (1, 1, 3), (2, 136, 70), (16, 512, 100), (17, 264, 33), (32, 1000, 64), (33, 72, 257),
         (64, 4104, 48), (65, 64, 64), (66, 1, 5), (100, 333, 129), (128, 128, 64), (129, 192, 65), (300, 200, 515),
         (1000, 520, 130), (4097, 64, 1030), (2050, 136, 4232),
         # the forms that the sizes above do not reach: two groups of 16 rows, 128 x 128 and 128 x 256 tiles
         (24, 72, 4500), (31, 1032, 4099), (1030, 72, 2063), (1024, 200, 2048), (4090, 72, 4090), (4096, 136, 4096),
         (923, 131, 3336), (909, 67, 3297), (1371, 8, 4804), (62, 2918, 3),
         (5975, 64, 644), (5970, 136, 645)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,F", GATED)
def test_gated_linear(cuda, M, D, F):
    g = gen(M * 7 + D + F, cuda)
    x, wg, wu = randn(g, M, D), randn(g, F, D, std=D**-0.5), randn(g, F, D, std=D**-0.5)
    for act, save in (("silu", True), ("gelu", False)):
        gated_check(x, wg, wu, act, ops.gated_linear(x, wg, wu, act, save=save), save)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("M,D,F", [(5, 96, 40), (200, 96, 72), (8200, 64, 1032)])
def test_gated_linear_activations(cuda, M, D, F, act):
    g = gen(3, cuda)
    x, wg, wu = randn(g, M, D, std=3.0), randn(g, F, D, std=D**-0.5), randn(g, F, D, std=D**-0.5)
    gated_check(x, wg, wu, act, ops.gated_linear(x, wg, wu, act, save=True), True)


# ---------------------------------------------------------------------------------------------------------------
# linear_i8
# ---------------------------------------------------------------------------------------------------------------
def i8_case(g, M, N, K, extreme=False):
    dev = g.device
    lo, hi = (-128, 128) if extreme else (-100, 101)
    x = torch.randint(lo, hi, (M, K), device=dev, generator=g).to(torch.int8)
    w = torch.randint(lo, hi, (N, K), device=dev, generator=g).to(torch.int8)
    if extreme:
        x[0].fill_(-128)
        w[0].fill_(-128)
    sx = torch.rand(M, device=dev, generator=g) * 0.05 + 1e-3
    sw = (torch.rand(N, device=dev, generator=g) * 0.05 + 1e-3) * K**-0.5
    return x, sx, w, sw, torch.randn(N, device=dev, generator=g)


def i8_check(x, sx, w, sw, b, act, y):
    z = (x.to(D64) @ w.to(D64).t()) * sx.to(D64)[:, None] * sw.to(D64)[None]
    mag = z.abs()
    if b is not None:
        z = z + b.to(D64)
        mag = mag + b.to(D64).abs()
    # int -> fp32, the scales' product, the scaling and the addition: one rounding each
    err = 4 * EPS_F32 * mag * 1.01
    f, _ = act64(z, act)
    err = err + (EPS_ACT * f.abs() if act == "tanh" else 0.0)
    eps = EPS_BF16 if y.dtype == torch.bfloat16 else EPS_F32
    within(y, f, err + eps * (f.abs() + err), "y")


I8 = [(1, 16, 16), (1, 1, 1), (3, 5, 7), (16, 100, 4096), (17, 33, 1000), (33, 64, 144), (64, 1000, 272), (65, 64, 128),
      (128, 128, 640), (130, 70, 130), (640, 1000, 512), (1030, 4100, 176), (4100, 4360, 144), (70, 17, 20000),
      (20, 6000, 500), (32, 4097, 4112), (1500, 1999, 400), (4090, 4090, 272), (4096, 4096, 100), (1870, 1110, 8), (3188, 1322, 8),
      (3468, 3641, 647),
      (4364, 2701, 130), (4361, 2704, 272)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", I8)
def test_linear_i8(cuda, M, N, K):
    g = gen(M + N + K, cuda)
    x, sx, w, sw, b = i8_case(g, M, N, K)
    i8_check(x, sx, w, sw, b, "none", ops.linear_i8(x, sx, w, sw, b))
    i8_check(x, sx, w, sw, None, "relu", ops.linear_i8(x, sx, w, sw, None, "relu", out_dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(4, 40, 131071), (80, 40, 131071)])
def test_linear_i8_longest_sum_is_exact(cuda, M, N, K):
    """K at its bound with -128 * -128 throughout: the largest 32-bit sum there is."""
    x, sx, w, sw, _ = i8_case(gen(1, cuda), M, N, K, extreme=True)
    sx, sw = torch.ones_like(sx), torch.ones_like(sw)
    y = ops.linear_i8(x, sx, w, sw, out_dtype=torch.float32)
    ref = x.to(D64) @ w.to(D64).t()
    assert ref[0, 0].item() == 131071 * 128 * 128
    assert torch.equal(y, ref.to(torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "tanh"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(5, 40, 96), (100, 72, 96), (2100, 2064, 64)])
def test_linear_i8_epilogues(cuda, M, N, K, out, act):
    x, sx, w, sw, b = i8_case(gen(5, cuda), M, N, K)
    i8_check(x, sx, w, sw, b, act, ops.linear_i8(x, sx, w, sw, b, act, out_dtype=out))


# ---------------------------------------------------------------------------------------------------------------
# gated_linear_bwd
# ---------------------------------------------------------------------------------------------------------------
def gated_bwd_check(dh, x, wg, wu, gate, up, act, out):
    DH, X, Wg, Wu, G, U = (t.to(D64) for t in (dh, x, wg, wu, gate, up))
    f, df = act64(G, act)
    # f and f' carry a few units in the last place of terms of size |f| + 1.13 and |G f''| <= 1
    dg, eg = DH * U * df, EPS_ACT * (DH * U).abs() * (1.13 + G.abs() * 2.0**-3)
    du, eu = DH * f, EPS_ACT * DH.abs() * (f.abs() + G.abs() * 2.0**-3)
    # the projections' gradients are rounded to bf16
    eg = eg + EPS_BF16 * (dg.abs() + eg) + 1e-38
    eu = eu + EPS_BF16 * (du.abs() + eu) + 1e-38
    M, F = dh.shape

    def one(got, ref, err, what):
        within(got, ref, err + EPS_BF16 * (ref.abs() + err) + 1e-38, what)

    mag = dg.abs() @ Wg.abs() + du.abs() @ Wu.abs()
    one(out[0], dg @ Wg + du @ Wu, eg @ Wg.abs() + eu @ Wu.abs() + 1.01 * (2 * F + 64) * EPS_SUM * mag, "dx")
    one(out[1], dg.t() @ X, eg.t() @ X.abs() + 1.01 * (M + 64) * EPS_SUM * (dg.abs().t() @ X.abs()), "dw_gate")
    one(out[2], du.t() @ X, eu.t() @ X.abs() + 1.01 * (M + 64) * EPS_SUM * (du.abs().t() @ X.abs()), "dw_up")


def gated_bwd_case(g, M, D, F, std=1.0):
    x, wg, wu = randn(g, M, D, std=std), randn(g, F, D, std=D**-0.5), randn(g, F, D, std=D**-0.5)
    gate, up = (x.float() @ wg.float().t()).bfloat16(), (x.float() @ wu.float().t()).bfloat16()
    return randn(g, M, F, std=0.1), x, wg, wu, gate, up


GATED_BWD = [(1, 64, 16), (1, 1, 1), (2, 136, 70), (3, 9, 1), (16, 512, 100), (17, 264, 33), (33, 72, 257), (64, 4104, 48),
             (64, 128, 3000), (65, 64, 64), (66, 1, 5), (100, 333, 129), (128, 128, 64), (129, 192, 65), (300, 200, 515),
             (1000, 520, 130), (4100, 64, 1030), (700, 4360, 4200),
             # every form and split of the two products
             (2634, 8, 2330), (1797, 185, 1), (2073, 16, 10), (36, 141, 2829), (2763, 4656, 1), (2178, 2144, 1),
             (33, 259, 2940), (34, 1808, 3272), (91, 10, 848), (55, 8, 1024), (33, 8, 2024), (129, 4208, 3876),
             (66, 2096, 1296), (66, 1028, 1520), (33, 1035, 2904), (2144, 1170, 1), (193, 4136, 2339), (66, 4240, 2081),
             (2078, 70, 1416), (67, 1048, 2845), (1870, 904, 1), (259, 3656, 2888), (2557, 1544, 2694), (8000, 520, 300),
             (8000, 1030, 520), (6000, 2056, 1024), (5550, 4728, 193), (5861, 522, 3385), (4130, 68, 2832),
             (5778, 136, 3466), (5704, 648, 3034), (5921, 646, 2808), (2787, 130, 3160),
             (7, 4104, 1030), (30, 2056, 1500), (5935, 131, 3777), (9, 640, 2000), (128, 1000, 777), (127, 1001, 777), (129, 1000, 777),
             # the products in one launch or in two, in every form, split and not
             (4209, 71, 1000), (3490, 329, 324), (1860, 2912, 874), (2249, 1769, 264), (474, 1988, 1488),
             (229, 3912, 1008), (395, 1488, 2648), (176, 4256, 1848), (368, 3112, 1224), (1189, 533, 5322),
             (3108, 2256, 219), (2541, 810, 3648), (5236, 2640, 169), (5923, 338, 5417),
             (1447, 3976, 832), (4861, 157, 4932), (223, 3984, 1437), (2589, 4016, 120), (68, 856, 5827),
             (770, 1000, 2700), (777, 1021, 2731), (4723, 1130, 539), (4012, 1328, 4943)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,F", GATED_BWD)
def test_gated_linear_bwd(cuda, M, D, F):
    case = gated_bwd_case(gen(M * 7 + D + F, cuda), M, D, F)
    gated_bwd_check(*case, "silu", ops.gated_linear_bwd(*case, "silu"))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("M,D,F", [(5, 96, 40), (200, 96, 72)])
def test_gated_linear_bwd_activations(cuda, M, D, F, act):
    case = gated_bwd_case(gen(9, cuda), M, D, F, std=3.0)
    gated_bwd_check(*case, act, ops.gated_linear_bwd(*case, act))


@pytest.mark.parametrize("act", ["none", "relu", "tanh", "silu", "gelu"])
def test_slopes_are_those_of_the_activations(act):
    """act64's slope, which the backward tests use, against differences in 64 bits."""
    v = torch.linspace(-9, 9, 2001, dtype=D64) + 1e-3
    h = 1e-5
    num = (act64(v + h, act)[0] - act64(v - h, act)[0]) / (2 * h)
    # third derivatives of all of them are below 4: h^2 / 6 * 4, and 2 roundings of values up to 9 over 2 h
    assert (num - act64(v, act)[1]).abs().max().item() < h * h + 9 * 2.0**-52 / h


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 200])
def test_tanh_slope_far_from_zero(cuda, M):
    """dG alone, one value a sum (Wg the identity, Wu zero): its relative error far out, where tanh itself is 1."""
    n = 64
    v = torch.linspace(0.1, 40.0, M * n, device=cuda).bfloat16().reshape(M, n)
    v[:, ::2] *= -1
    eye, none = torch.eye(n, device=cuda).bfloat16(), torch.zeros(n, n, device=cuda).bfloat16()
    one = torch.ones(M, n, device=cuda).bfloat16()
    dx, _, _ = ops.gated_linear_bwd(one, none[:1].expand(M, n), eye, none, v, one, "tanh")
    ref = 1 / torch.cosh(v.to(D64)) ** 2
    # the exponent 2 |v| log2(e) of up to 116 has two roundings (its factor's and its own), 2^-23 of ln 2 times it;
    # exp2, the reciprocal and the products a few units of 2^-24; below 0.7 a tanh off by 5 of them, squared and taken
    # from 1 to no less than 0.63; two roundings to bf16, dG's and dX's
    rel = 2.0**-23 * 2 * v.to(D64).abs() + 32 * EPS_F32
    assert (((dx.to(D64) - ref).abs() / ref) <= rel + 2.02 * EPS_BF16).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "tanh"])
def test_gated_gradient_against_differences(cuda, act):
    """The whole backward pass against differences of the forward definition in 64 bits."""
    g = gen(11, cuda)
    M, D, F = 6, 24, 40
    x, wg, wu = randn(g, M, D), randn(g, F, D, std=0.3), randn(g, F, D, std=0.3)
    _, gate, up = ops.gated_linear(x, wg, wu, act, save=True)
    dh = randn(g, M, F)
    got = ops.gated_linear_bwd(dh, x, wg, wu, gate, up, act)
    leaves = [t.to(D64) for t in (x, wg, wu)]

    def value(x, wg, wu):
        return (dh.to(D64) * act64(x @ wg.t(), act)[0] * (x @ wu.t())).sum().item()

    h = 1e-6
    for i, leaf in enumerate(leaves):
        for _ in range(12):
            at = tuple(int(torch.randint(n, (1,), device=cuda, generator=g)) for n in leaf.shape)
            side = []
            for sign in (1, -1):
                moved = [t.clone() for t in leaves]
                moved[i][at] += sign * h
                side.append(value(*moved))
            num = (side[0] - side[1]) / (2 * h)
            # saved projections, dG / dU and the gradient itself are rounded to bf16: each term of the sums is off by
            # at most 2^-8 for dG / dU, and by 2^-8 of its projections' size (|f''| <= 1.6) for the saved ones
            dxs, a, b = dh.to(D64), leaves[0] @ leaves[1].t(), leaves[0] @ leaves[2].t()
            f, df = act64(a, act)
            tg = EPS_BF16 * dxs.abs() * ((b * df).abs() * 2 + b.abs() * 1.6 * a.abs())
            tu = EPS_BF16 * dxs.abs() * (f.abs() + 1.13 * a.abs())
            bound = {0: tg @ leaves[1].abs() + tu @ leaves[2].abs(), 1: tg.t() @ leaves[0].abs(),
                     2: tu.t() @ leaves[0].abs()}[i][at].item()
            assert abs(got[i][at].item() - num) <= 1.05 * bound + EPS_BF16 * abs(num) + 1e-6, (i, at)


# ---------------------------------------------------------------------------------------------------------------
# rmsnorm_i8
# ---------------------------------------------------------------------------------------------------------------
def norm_check(x, w, r, eps, out):
    q, scale, s = out
    v = x.to(D64) + (r.to(D64) if r is not None else 0.0)
    D = x.shape[1]
    y = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w.to(D64)
    # the fp32 sum v has one rounding; the mean's D additions weigh half in the root
    rel = EPS_F32 * 8 + D * EPS_F32 * 0.5
    top = y.abs().amax(1)
    within(scale, top / 127, rel * top / 127 + 1e-45, "scale")
    if r is not None:
        eps_s = EPS_BF16 if s.dtype == torch.bfloat16 else EPS_F32
        within(s, v, 1.01 * eps_s * v.abs() + EPS_F32 * v.abs() + 1e-38, "s")
    else:
        assert s is x
    # q: the nearest integer of y / scale, whose own error is a few 2^-24 of at most 127
    z = y / (top / 127).clamp(min=1e-300)[:, None]
    assert (q.to(D64) - z).abs().max().item() <= 0.5 + 127 * 8 * EPS_F32
    # (the factor 1 / rms cancels in q: no error of the mean in it)
    assert q.to(torch.int32).abs().max().item() <= 127


NORM = [(1, 1), (1, 8), (3, 7), (5, 64), (4, 512), (9, 513), (2, 1000), (7, 1024), (3, 1025), (2, 2048), (3, 2056), (1, 4096),
        (33, 4100), (3, 8192), (2, 8193), (2, 16384), (3, 20001), (2, 32768), (1000, 96), (20000, 17)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,D", NORM)
def test_rmsnorm_i8(cuda, M, D, dtype):
    g = gen(M + D, cuda)
    x, r = randn(g, M, D, dtype=dtype), randn(g, M, D, std=5.0, dtype=dtype)
    w = (1 + 0.2 * torch.randn(D, device=cuda, generator=g)).to(dtype)
    norm_check(x, w, r, 1e-6, ops.rmsnorm_i8(x, w, r))
    norm_check(x, w, None, 1e-5, ops.rmsnorm_i8(x, w, eps=1e-5))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [100, 3000, 16000])
def test_rmsnorm_i8_special_rows(cuda, D):
    """Rows of zeros, of values that are not finite, of tiny and of huge ones; no row touches another."""
    g = gen(2, cuda)
    x = randn(g, 9, D, dtype=torch.float32)
    x[0] = 0
    x[2, D // 2] = float("nan")
    x[3, 1] = float("inf")
    x[4, D - 1] = -float("inf")
    x[5] *= 1e-30
    x[6] *= 1e18 / D**0.5
    x[7] *= 1e30  # the squares overflow
    w = torch.ones(D, device=cuda)
    q, scale, s = ops.rmsnorm_i8(x, w, torch.zeros_like(x))
    assert torch.equal(s.isnan(), x.isnan()) and torch.equal(s.nan_to_num(), x.nan_to_num())
    assert scale[0].item() == 0 and not q[0].any()
    for row in (2, 3, 4, 7):
        assert math.isnan(scale[row].item()) and not q[row].any(), row
    for row in (1, 5, 6, 8):
        one = ops.rmsnorm_i8(x[row : row + 1], w)
        v = x[row : row + 1]
        norm_check(v, w, None, 1e-6, ops.rmsnorm_i8(v, w))
        assert torch.equal(one[0][0], q[row]) and torch.equal(one[1][0], scale[row]), row


# ---------------------------------------------------------------------------------------------------------------
# distill_kl
# ---------------------------------------------------------------------------------------------------------------
def distill64(z, tv, ti, T, scale):
    """(dz, loss, p, log terms' size) in 64 bits."""
    M, N = z.shape
    logp = torch.log_softmax(z.to(D64) / T, 1)
    there = (ti >= 0) & (ti < N) & (tv != -math.inf)
    some = there.any(1, keepdim=True)
    t = torch.where(there, tv.to(D64) / T, torch.full_like(tv, -math.inf, dtype=D64))
    t = torch.where(some, t, torch.zeros_like(t))
    logq = torch.log_softmax(t, 1)
    q = torch.where(there, torch.exp(logq), torch.zeros_like(logq))
    at = torch.where(there, ti.long(), torch.zeros_like(ti.long()))
    lp = logp.gather(1, at)
    terms = torch.where(q > 0, q * (torch.where(q > 0, logq, torch.zeros_like(logq)) - lp), torch.zeros_like(q))
    p = torch.exp(logp)
    sq = torch.zeros_like(p).scatter_add_(1, at, q)
    dz = torch.where(some, scale * T * (p - sq), torch.zeros_like(p))
    size = torch.where(q > 0, q * (logq.abs() + lp.abs()), torch.zeros_like(q)).sum(1)
    return dz, T * T * terms.sum(1), p, sq, T * T * size


def distill_check(z, tv, ti, T, scale, dz, loss):
    ref, rl, p, sq, size = distill64(z, tv, ti, T, scale)
    zf = z.to(D64)
    N = z.shape[1]
    zmax = zf.amax(1, keepdim=True)
    # exponent (z - max) log2(e) / T: three roundings of its size; the sum of N terms in at most N / 64 + 64 steps
    # that do not cancel; exp2, the division and the products a few units
    arg = torch.where(torch.isfinite(zf), (zmax - zf) / T, torch.zeros_like(zf))
    rel_e = EPS_F32 * (4 * arg + 8)
    rel_s = (p * rel_e).sum(1, keepdim=True) + EPS_F32 * (N / 64 + 64)
    if dz is not None:
        err = scale * T * (p * (rel_e + rel_s) + sq * 64 * EPS_F32)
        eps = EPS_BF16 if dz.dtype == torch.bfloat16 else EPS_F32
        within(dz, ref, err + 1.01 * eps * (ref.abs() + err) + 1e-38, "dz")
    K = tv.shape[1]
    lerr = (64 + K) * EPS_F32 * size + T * T * (rel_s[:, 0] + EPS_F32 * 8 * (zmax.abs()[:, 0] / T + 1))
    within(loss, rl, lerr + 1e-38, "loss")


def distill_case(g, M, N, K, dtype=torch.float32, index=torch.int64, std=2.0):
    dev = g.device
    z = randn(g, M, N, std=std, dtype=dtype)
    tv = randn(g, M, K, std=3.0, dtype=dtype)
    ti = torch.randint(0, N, (M, K), device=dev, generator=g).to(index)
    drop = torch.rand(M, K, device=dev, generator=g) < 0.2
    ti[drop] = -1
    return z, tv, ti


DISTILL = [(1, 1, 1), (1, 10, 3), (3, 2, 2), (5, 100, 10), (640, 1000, 10), (9, 1017, 64), (4, 1018, 5), (3, 4089, 33),
           (2, 4090, 7), (3, 8185, 16), (2, 8186, 1), (130, 16377, 12), (129, 16378, 12), (130, 32770, 20), (3, 50001, 64),
           (131, 65001, 9), (130, 65529, 9), (129, 65530, 9), (1, 131072, 40), (140, 131065, 5), (2, 250001, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", DISTILL)
def test_distill_kl(cuda, M, N, K, dtype):
    z, tv, ti = distill_case(gen(M + N + K, cuda), M, N, K, dtype)
    dz, loss = ops.distill_kl(z, tv, ti, temperature=2.0, scale=0.5)
    assert dz.dtype == dtype
    distill_check(z, tv, ti, 2.0, 0.5, dz, loss)
    none, alone = ops.distill_kl(z, tv, ti, temperature=2.0, grad=False)
    assert none is None and torch.equal(alone, loss)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(70, 37, 1024), (3, 5000, 1024), (2, 70000, 700)])
def test_distill_kl_many_entries_and_types(cuda, M, N, K):
    """Classes that occur many times add up; int32 classes, other types of teacher and gradient."""
    z, tv, ti = distill_case(gen(1, cuda), M, N, K, torch.bfloat16, torch.int32)
    dz, loss = ops.distill_kl(z, tv.float(), ti, grad_dtype=torch.float32)
    assert dz.dtype == torch.float32
    # a sum of up to K shares of one class
    ref, rl, p, sq, size = distill64(z, tv.float(), ti, 1.0, 1.0)
    assert (dz.to(D64) - ref).abs().max().item() < (K + 200) * EPS_F32
    distill_check(z, tv.float(), ti, 1.0, 1.0, None, loss)
    again = ops.distill_kl(z, tv.float(), ti, grad_dtype=torch.float32)
    assert torch.equal(dz, again[0]) and torch.equal(loss, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("N", [50, 3000, 20000, 40000, 140000])
def test_distill_kl_masks(cuda, N):
    """Rows without entries, entries out of range or of -inf, masked classes, the type's lowest value."""
    low = torch.finfo(torch.float32).min
    z, tv, ti = distill_case(gen(4, cuda), 9, N, 6)
    ti = torch.where(ti < 0, ti + 1, ti)  # all there
    ti[0] = -1
    ti[1] = torch.tensor([N, -7, 2**40, -(2**40), N + 1, -1], device=cuda)
    tv[2] = -math.inf
    tv[3, :5] = -math.inf
    tv[4, ::2] = low
    tv[5] = low
    z[6, : N // 2] = -math.inf
    ti[6] = N - 1 - torch.arange(6, device=cuda)
    z[7, : N // 2] = low
    z[3] = low  # nothing but the lowest value: even odds
    ti[7] = N - 1 - torch.arange(6, device=cuda)
    tv[8, 3] = float("nan")
    ti[8, 3] = -1  # a NaN that is not there
    dz, loss = ops.distill_kl(z, tv, ti, temperature=1.5)
    for row in (0, 1, 2):
        assert loss[row].item() == 0 and not dz[row].any(), row
    tv[8, 3] = 0.0
    distill_check(z[3:], tv[3:], ti[3:], 1.5, 1.0, dz[3:], loss[3:])


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-3e4, 1e6])
def test_distill_kl_logits_far_from_zero(cuda, shift):
    """A row's logits count by their differences alone (here exact: multiples of 1/4 below 2^24 / 4)."""
    g = gen(8, cuda)
    z = torch.randint(-40, 40, (5, 3001), device=cuda, generator=g) / 4.0
    tv = torch.randint(-40, 40, (5, 7), device=cuda, generator=g) / 4.0
    ti = torch.randint(0, 3001, (5, 7), device=cuda, generator=g)
    a, b = ops.distill_kl(z, tv, ti, temperature=2.0), ops.distill_kl(z + shift, tv + shift, ti, temperature=2.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("N,pad", [(1000, 3), (20000, 5), (40001, 8), (150000, 1)])
def test_distill_kl_strided_logits(cuda, N, pad):
    """Rows of a wider matrix, another pitch than the gradient's and a start that is not aligned."""
    g = gen(8, cuda)
    z, tv, ti = distill_case(g, 3, N + pad, 9, torch.bfloat16)
    ti = ti.clamp(max=N - 1)
    view = z[:, pad // 2 : pad // 2 + N]
    a, b = ops.distill_kl(view, tv, ti), ops.distill_kl(view.contiguous(), tv, ti)
    distill_check(view, tv, ti, 1.0, 1.0, a[0], a[1])
    distill_check(view, tv, ti, 1.0, 1.0, b[0], b[1])


@pytest.mark.gpu
def test_distill_kl_no_entries_at_all(cuda):
    z = randn(gen(1, cuda), 4, 100)
    dz, loss = ops.distill_kl(z, torch.empty(4, 0, device=cuda), torch.empty(4, 0, dtype=torch.int64, device=cuda))
    assert not dz.any() and not loss.any()


@pytest.mark.gpu
def test_distill_gradient_against_differences(cuda):
    g = gen(6, cuda)
    z, tv, ti = distill_case(g, 3, 40, 8)
    T = 2.0
    dz, _ = ops.distill_kl(z, tv, ti, temperature=T, scale=0.25)
    h = 1e-5
    for _ in range(30):
        at = (int(torch.randint(3, (1,), device=cuda, generator=g)), int(torch.randint(40, (1,), device=cuda, generator=g)))
        side = []
        for sign in (1, -1):
            m = z.to(D64)
            m[at] += sign * h
            side.append(0.25 * distill64(m, tv, ti, T, 1.0)[1].sum().item())
        num = (side[0] - side[1]) / (2 * h)
        # h^2 / 6 of a third derivative below 1, the differences' rounding, and fp32 in the kernel
        assert abs(dz[at].item() - num) < h * h + 1e-15 / h * 100 + 1e-6


# ---------------------------------------------------------------------------------------------------------------
# strides, streams, graphs, a run of them together
# ---------------------------------------------------------------------------------------------------------------
def wide_view(t, left, right):
    """t's values as columns of a wider matrix whose other columns are NaN (127 for int8)."""
    rows, cols = t.shape
    fill = 127 if t.dtype == torch.int8 else float("nan")
    big = torch.full((rows, left + cols + right), fill, dtype=t.dtype, device=t.device)
    view = big[:, left : left + cols]
    view.copy_(t)
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("left,right", [(0, 8), (8, 8), (3, 0), (1, 4)])
@pytest.mark.parametrize("M,D,F", [(3, 72, 40), (20, 64, 4500), (150, 104, 200), (90, 100, 130)])
def test_gated_linear_strided(cuda, M, D, F, left, right):
    case = gated_bwd_case(gen(4, cuda), M, D, F)
    dh, x, wg, wu, gate, up = case
    v = [wide_view(t, left, right) for t in case]
    gated_check(x, wg, wu, "silu", ops.gated_linear(v[1], v[2], v[3], "silu", save=True), True)
    gated_bwd_check(*case, "silu", ops.gated_linear_bwd(*v, "silu"))
    # the two weights of one pitch each, a transposed input
    xt = x.t().contiguous().t()
    gated_check(x, wg, wu, "silu", ops.gated_linear(xt, wg, v[3], "silu", save=True), True)
    gated_bwd_check(*case, "silu", ops.gated_linear_bwd(dh.t().contiguous().t(), xt, v[2], wu, gate, v[5], "silu"))
    # one row of x for all tokens
    same = x[:1].expand(M, D)
    gated_check(same, wg, wu, "silu", ops.gated_linear(same, wg, wu, "silu"), False)


@pytest.mark.gpu
@pytest.mark.parametrize("left,right", [(0, 16), (16, 16), (3, 0)])
@pytest.mark.parametrize("M,N,K", [(3, 40, 96), (200, 130, 96), (90, 33, 100)])
def test_linear_i8_strided(cuda, M, N, K, left, right):
    x, sx, w, sw, b = i8_case(gen(4, cuda), M, N, K)
    sx2, sw2, b2 = (torch.stack([t, torch.full_like(t, float("nan"))], 1)[:, 0] for t in (sx, sw, b))
    i8_check(x, sx, w, sw, b, "none", ops.linear_i8(wide_view(x, left, right), sx2, wide_view(w, left, right), sw2, b2))


@pytest.mark.gpu
@pytest.mark.parametrize("left", range(0, 17, 2))
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 5, 7), (3, 2, 17), (40, 7, 31), (5, 300, 455)])
def test_linear_i8_rows_of_any_alignment(cuda, M, N, K, left):
    x, sx, w, sw, b = i8_case(gen(6, cuda), M, N, K)
    want = ops.linear_i8(x, sx, w, sw, b)
    i8_check(x, sx, w, sw, b, "none", want)
    got = ops.linear_i8(wide_view(x, left, left % 3), sx, wide_view(w, left + 1, left % 5), sw, b)
    assert torch.equal(got, want)
    # columns of a transposed matrix, and one row for all
    assert torch.equal(ops.linear_i8(x.t().contiguous().t(), sx, w, sw, b), want)
    same = w[:1].expand(N, K)
    i8_check(x, sx, same, sw, b, "none", ops.linear_i8(x, sx, same, sw, b))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(65, 70, 9000), (152, 1024, 7248), (90, 33, 15608), (300, 129, 4100), (3, 64, 16000),
                                   (33, 1, 5001), (128, 520, 16383)])
def test_few_tiles_of_long_rows(cuda, M, N, K):
    """Products that are split over K: every epilogue."""
    g = gen(K, cuda)
    x, sx, w, sw, b = i8_case(g, M, N, K)
    for act, out in (("none", torch.float32), ("relu", torch.bfloat16), ("tanh", torch.float32)):
        y = ops.linear_i8(x, sx, w, sw, b, act, out_dtype=out)
        i8_check(x, sx, w, sw, b, act, y)
        assert torch.equal(y, ops.linear_i8(x, sx, w, sw, b, act, out_dtype=out))
    i8_check(x, sx, w, sw, None, "none", ops.linear_i8(x, sx, w, sw))
    _, x, wg, wu, _, _ = gated_bwd_case(g, M, K, N)
    for act in ("none", "silu", "gelu", "tanh", "relu"):
        gated_check(x, wg, wu, act, ops.gated_linear(x, wg, wu, act, save=True), True)
    gated_check(x, wg, wu, "silu", ops.gated_linear(x, wg, wu, "silu"), False)


def test_workspaces():
    """Split products of few tiles alone ask for a workspace."""
    K = ops.feedforward._K
    assert K.gated_forward_bytes(152, 7248, 1024) > 0 and K.linear_i8_bytes(90, 960, 15608) > 0
    for M, D, F in ((1, 4096, 8192), (777, 1024, 2731), (8192, 4096, 12288), (1, 1, 1), (64, 64, 64)):
        assert K.gated_forward_bytes(M, D, F) == 0 and K.linear_i8_bytes(M, F, D) == 0
    # what the wrappers do not ask for is never split
    for M, F in ((1, 64), (33, 100), (200, 200), (64, 1 << 14), (1024, 1025), (1 << 14, 65), (1, 1 << 20)):
        for k in (*range(2020, 2048), 100):
            assert K.gated_forward_bytes(M, k, F) == 0
        for k in (*range(4070, 4096), 100):
            assert K.linear_i8_bytes(M, F, k) == 0
    for M, F in ((16, 64), (1, 5000), (1024, 1025), (1 << 14, 65), (1, (1 << 20) + 1), ((1 << 20) + 1, 1), (300, 3500)):
        for k in (4097, 20000, 131071):
            assert K.gated_forward_bytes(M, k, F) == 0 and K.linear_i8_bytes(M, F, k) == 0
    with pytest.raises(ops.feedforward._C.MccError):
        K.gated_forward(152, 7248, 1024, 0, 0, 7248, 0, 0, 7248, 0)
    with pytest.raises(ops.feedforward._C.MccError):
        K.linear_i8(90, 960, 15616, 0, 0, 15616, 0, 0, 15616, 0, 0, 0, False)


@pytest.mark.gpu
@pytest.mark.parametrize("left", [0, 1, 2, 5, 7])
@pytest.mark.parametrize("K", [1, 7, 9, 15, 17, 127, 455, 2055, 4099, 6185])
@pytest.mark.parametrize("M", [1, 16, 20, 32, 33])
def test_few_rows_of_any_alignment(cuda, M, K, left):
    x, sx, w, sw, b = i8_case(gen(K, cuda), M, 50, K)
    i8_check(x, sx, w, sw, b, "none", ops.linear_i8(wide_view(x, left, 0), sx, wide_view(w, left + 1, 2), sw, b))
    _, x, wg, wu, _, _ = gated_bwd_case(gen(K, cuda), M, K, 35)
    out = ops.gated_linear(wide_view(x, left, 1), wide_view(wg, left, 0), wide_view(wu, left + 1, 2), "silu", save=True)
    gated_check(x, wg, wu, "silu", out, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("left,right", [(0, 8), (8, 8), (3, 0)])
@pytest.mark.parametrize("M,D", [(5, 96), (3, 4096), (2, 10007)])
def test_rmsnorm_i8_strided(cuda, M, D, left, right, dtype):
    g = gen(4, cuda)
    x, r = randn(g, M, D, dtype=dtype), randn(g, M, D, dtype=dtype)
    w = randn(g, D, dtype=dtype)
    norm_check(x, w, r, 1e-6, ops.rmsnorm_i8(wide_view(x, left, right), torch.stack([w, w], 1)[:, 0],
                                             wide_view(r, left, right)))


@pytest.mark.gpu
def test_empty_batches(cuda):
    g = gen(1, cuda)
    x, wg = randn(g, 0, 64), randn(g, 32, 64)
    h, gate, up = ops.gated_linear(x, wg, wg, save=True)
    assert h.shape == gate.shape == up.shape == (0, 32)
    dx, dwg, dwu = ops.gated_linear_bwd(h, x, wg, wg, gate, up)
    assert dx.shape == (0, 64) and not dwg.any() and not dwu.any() and dwg.shape == dwu.shape == (32, 64)
    q, s, v = ops.rmsnorm_i8(x, wg[0], x)
    assert q.shape == v.shape == (0, 64) and s.shape == (0,)
    wq, sw = torch.ones(8, 64, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)
    assert ops.linear_i8(q, s, wq, sw).shape == (0, 8)
    dz, loss = ops.distill_kl(x, torch.empty(0, 3, device=cuda), torch.empty(0, 3, dtype=torch.int64, device=cuda))
    assert dz.shape == (0, 64) and loss.shape == (0,)


@pytest.mark.gpu
def test_rmsnorm_i8_without_eps(cuda):
    """eps = 0: a row of zeros has scale 0, a row whose squares underflow is NaN, others are as they were."""
    g = gen(5, cuda)
    x, w = randn(g, 6, 320, dtype=torch.float32), randn(g, 320, dtype=torch.float32)
    x[1] = 0
    x[3] *= 1e-30
    q, scale, _ = ops.rmsnorm_i8(x, w, eps=0.0)
    assert scale[1].item() == 0 and not q[1].any()
    assert math.isnan(scale[3].item()) and not q[3].any()
    rows = [0, 2, 4, 5]
    v = x[rows]
    norm_check(v, w, None, 0.0, (q[rows], scale[rows], v))


@pytest.mark.gpu
def test_many_short_rows(cuda):
    """More rows than 65535 groups of 16."""
    g = gen(6, cuda)
    M = 1_100_003
    case = gated_bwd_case(g, M, 24, 8)
    gated_check(*case[1:4], "silu", ops.gated_linear(*case[1:4], "silu", save=True), True)
    gated_bwd_check(*case, "silu", ops.gated_linear_bwd(*case, "silu"))
    x, sx, w, sw, b = i8_case(g, M, 7, 40)
    i8_check(x, sx, w, sw, b, "relu", ops.linear_i8(x, sx, w, sw, b, "relu"))
    x, w = randn(g, M, 10), randn(g, 10)
    norm_check(x, w, x, 1e-6, ops.rmsnorm_i8(x, w, x))
    z, tv, ti = distill_case(g, M, 5, 2)
    distill_check(z, tv, ti, 1.0, 1.0, *ops.distill_kl(z, tv, ti))


def spread(M, cuda):
    """Rows of a large matrix, the first and the last among them."""
    return torch.tensor([0, 1, M // 3, M // 2, M - 130, M - 2, M - 1], device=cuda)


@pytest.mark.gpu
def test_matrices_past_32_bits(cuda):
    """Matrices of more than 2^31 values: what rows far behind hold."""
    g = gen(7, cuda)
    M, F, D = 70_001, 32_768, 8
    at = spread(M, cuda)
    x, wg, wu = randn(g, M, D), randn(g, F, D), randn(g, F, D)
    h, gate, up = ops.gated_linear(x, wg, wu, "silu", save=True)
    gated_check(x[at], wg, wu, "silu", (h[at], gate[at], up[at]), True)
    # gradients of these rows alone, the others' are zeros
    h.zero_()
    h[at] = randn(g, at.numel(), F, std=0.1)
    dx, dwg, dwu = ops.gated_linear_bwd(h, x, wg, wu, gate, up, "silu")
    gated_bwd_check(h[at], x[at], wg, wu, gate[at], up[at], "silu", (dx[at], dwg, dwu))
    dx[at] = 0
    assert not dx.any()
    del h, gate, up, dx, dwg, dwu
    F = F + 1  # (rows of any alignment)
    x, sx, w, sw, b = i8_case(g, M, F, 16)
    i8_check(x[at], sx[at], w, sw, b, "none", ops.linear_i8(x, sx, w, sw, b)[at])


@pytest.mark.gpu
def test_rows_past_32_bits(cuda):
    g = gen(8, cuda)
    M, D = 70_001, 32_767
    at = spread(M, cuda)
    x, w = randn(g, M, D), randn(g, D)
    q, scale, s = ops.rmsnorm_i8(x, w, x)
    norm_check(x[at], w, x[at], 1e-6, (q[at], scale[at], s[at]))
    del q, scale, s
    _, tv, ti = distill_case(g, M, 50, 3)
    dz, loss = ops.distill_kl(x, tv, ti)
    distill_check(x[at], tv[at], ti[at], 1.0, 1.0, dz[at], loss[at])


def serving(x, r, w, w1, s1, b1):
    """A quantised projection behind its norm."""
    q, s, v = ops.rmsnorm_i8(x, w, r)
    return ops.linear_i8(q, s, w1, s1, b1, "relu"), v


def training(x, wg, wu, head, tv, ti):
    """A student's gated block and head on a teacher's top logits: every gradient, and the loss."""
    h, gate, up = ops.gated_linear(x, wg, wu, "silu", save=True)
    z = ops.linear(h, head)
    dz, loss = ops.distill_kl(z, tv, ti, temperature=2.0, scale=1.0 / x.shape[0])
    dhead, _ = ops.linear_wgrad(dz, h)
    dh = ops.linear_dgrad(dz, head)
    dx, dwg, dwu = ops.gated_linear_bwd(dh, x, wg, wu, gate, up, "silu")
    return [loss, dx, dwg, dwu, dhead]


def training_case(g, M=200, D=96, F=160, N=104, K=8):
    z, tv, ti = distill_case(g, M, N, K)
    return (randn(g, M, D), randn(g, F, D, std=D**-0.5), randn(g, F, D, std=D**-0.5), randn(g, N, F, std=F**-0.5), tv, ti)


@pytest.mark.gpu
def test_training_run_against_autograd(cuda):
    """The chain's gradients against torch's own derivative of the same chain in 64 bits.  Nine roundings to bf16 lie on
    the longest way (h, z, dz, dh, gate, up, dG, dU, the gradient): each moves a sum of independent terms by at most
    2^-8 of its terms' root sum of squares, so the whole gradient by at most 9 * 2^-8 of its norm times what
    cancellation in the steps between costs (a factor of 3 here: |p - q| is about a third of |p| + |q|)."""
    x, wg, wu, head, tv, ti = training_case(gen(3, cuda))
    got = training(x, wg, wu, head, tv, ti)
    leaf = [t.to(D64).requires_grad_() for t in (x, wg, wu, head)]
    h = torch.nn.functional.silu(leaf[0] @ leaf[1].t()) * (leaf[0] @ leaf[2].t())
    loss = distill64(h @ leaf[3].t(), tv, ti, 2.0, 1.0)[1]
    (loss.sum() / x.shape[0]).backward()
    assert ((got[0] - loss.detach()).abs() <= 2.0**-5 * (loss.detach().abs() + 1)).all()
    for a, b in zip(got[1:], leaf):
        rel = ((a.to(D64) - b.grad).norm() / b.grad.norm()).item()
        assert rel < 27 * 2.0**-8, rel


@pytest.mark.gpu
def test_serving_run(cuda):
    g = gen(3, cuda)
    M, D, N = 70, 256, 120
    x, r, w = randn(g, M, D), randn(g, M, D), randn(g, D)
    _, _, w1, s1, b1 = i8_case(g, 1, N, D)
    y, v = serving(x, r, w, w1, s1, b1)
    s = x.to(D64) + r.to(D64)
    n = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * w.to(D64)
    W = w1.to(D64) * s1.to(D64)[:, None]
    ref = n @ W.t() + b1.to(D64)
    # quantising moves every value by at most half a step
    err = (n.abs().amax(1, keepdim=True) / 127 * (0.5 + 1e-3)) @ W.abs().sum(1)[None, :]
    within(y, ref.clamp(min=0), err + EPS_BF16 * (ref.abs() + err) + 1e-6, "y")
    assert torch.equal(v, (x.float() + r.float()).bfloat16())


@pytest.mark.gpu
def test_runs_repeat_exactly_on_any_stream(cuda):
    """The same bits again, on another stream, and from two streams at once."""
    case, big = training_case(gen(3, cuda)), training_case(gen(4, cuda), 700, 520, 1000, 3000, 16)
    for c in (case, big):
        one = training(*c)
        for a, b in zip(one, training(*c)):
            assert torch.equal(a, b)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        out = {}
        for rep in range(3):
            for s in (s1, s2):
                with torch.cuda.stream(s):
                    out[s] = training(*c)
        torch.cuda.synchronize()
        for s in (s1, s2):
            for a, b in zip(one, out[s]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_runs(cuda):
    """Training and serving runs captured into two graphs, replayed in turn with new inputs and eager work between."""
    g = gen(5, cuda)
    t_in = [t.clone() for t in training_case(g)]
    s_in = [randn(g, 9, 256), randn(g, 9, 256), randn(g, 256), *i8_case(g, 1, 120, 256)[2:]]
    rows_in = gated_bwd_case(g, 7, 136, 520)  # few rows: other kernels than t_in's
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        training(*t_in), serving(*s_in), ops.gated_linear_bwd(*rows_in)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = training(*t_in)
    with torch.cuda.graph(g2):
        o2 = [*serving(*s_in), *ops.gated_linear_bwd(*rows_in)]
    for rep in range(4):
        new = training_case(gen(10 + rep, cuda))
        for a, b in zip(t_in, new):
            a.copy_(b)
        s_in[0].copy_(randn(gen(20 + rep, cuda), 9, 256))
        rows_in[0].copy_(randn(gen(30 + rep, cuda), 7, 520))
        g1.replay()
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        for a, b in zip(o1, training(*t_in)):
            assert torch.equal(a, b), rep
        for a, b in zip(o2, [*serving(*s_in), *ops.gated_linear_bwd(*rows_in)]):
            assert torch.equal(a, b), rep


# ---------------------------------------------------------------------------------------------------------------
# several operands of one call whose columns are not next to each other
# ---------------------------------------------------------------------------------------------------------------
def across(t):
    """t's values, its columns a row's length apart."""
    return t.t().contiguous().t()


@pytest.mark.parametrize("M,D,F", [(300, 1024, 512), (2048, 512, 1024), (40, 100, 60), (64, 7, 64), (20, 64, 64), (20, 65, 64)])
def test_copies_of_several_operands(monkeypatch, M, D, F):
    """What is copied for one call lies in places of its own until the copying kernel has been launched."""
    ff = ops.feedforward
    todo = []

    def launch(dev, fn, ms):
        spans = sorted((a, a + (rows - 1) * pitch + cols) for src, dst, ld, ldd, rows, cols in ms
                       for a, pitch in ((src, ld), (dst, ldd)))
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), spans
        for src, dst, ld, ldd, rows, cols in ms:
            ctypes.memset(dst, 0, rows * ldd)
            for r in range(rows):
                ctypes.memmove(dst + r * ldd, src + r * ld, cols)
        todo.extend(ms)

    monkeypatch.setattr(ff, "_run", launch)
    g = torch.Generator().manual_seed(M)
    ts = [torch.randn(M, D, generator=g).bfloat16(), *(across(torch.randn(F, D, generator=g).bfloat16()) for _ in range(2))]
    for x in (ts[0], across(ts[0])):
        *got, any_ = ff._pieces(torch.device("cpu"), 8, x, ts[1], ts[2])
        for (t, ld), want in zip(got, ts):
            assert t.stride() == (ld, 1) and torch.equal(t[:, :D], want) and (any_ or not t[:, D:].any())
            assert any_ or (ld % 8 == 0 and t.data_ptr() % 16 == 0)
    assert bool(todo) == (M > 32 and D % 8 != 0)  # (a dense copy of whole pieces is not copied again)


@pytest.mark.parametrize("n,dtype", [(8, torch.bfloat16), (16, torch.int8)])
@pytest.mark.parametrize("M", [1, 32])
def test_few_rows_alone_are_copied_for_large_weights(monkeypatch, M, n, dtype):
    """Large weights of whole pieces are read as such whatever x's alignment."""
    ff = ops.feedforward
    todo = []
    monkeypatch.setattr(ff, "_run", lambda dev, fn, ms: todo.append(ms))
    size = 16 // n
    for K, N, copied in ((16384, 64, True), (4096, 1 << 13, True), (1024, 512, False)):
        K //= size  # (a row of K bytes)
        x, w = torch.zeros(M, K + 8, dtype=dtype)[:, 1 : K + 1], torch.zeros(N, K, dtype=dtype)
        todo.clear()
        (xa, ldx), (wa, ldw), any_ = ff._pieces(torch.device("cpu"), n, x, w)
        assert wa is w and ldw == K and any_ is not copied
        assert len(todo) == copied and (not copied or (len(todo[0]) == 1 and todo[0][0][0] == x.data_ptr() and xa is not x))
        # whole pieces throughout: nothing to do; weights that are not: as they are
        assert ff._pieces(torch.device("cpu"), n, w[:M], w)[2] is False and len(todo) == copied
        v = torch.zeros(N, K + 8, dtype=dtype)[:, 1 : K + 1]
        assert ff._pieces(torch.device("cpu"), n, x, v)[2] is True and len(todo) == copied


@pytest.mark.gpu
@pytest.mark.parametrize("left", [1, 5])
@pytest.mark.parametrize("M,D,F", [(1, 4096, 8200), (32, 4096, 4099), (7, 16384, 33), (20, 8192, 70), (17, 512, 100)])
def test_few_rows_of_another_alignment_than_the_weights(cuda, M, D, F, left):
    g = gen(M + D, cuda)
    _, x, wg, wu, _, _ = gated_bwd_case(g, M, D, F)
    gated_check(x, wg, wu, "silu", ops.gated_linear(wide_view(x, left, 2), wg, wu, "silu", save=True), True)
    xq, sx, wq, sw, b = i8_case(g, M, F, D)
    i8_check(xq, sx, wq, sw, b, "none", ops.linear_i8(wide_view(xq, left, 2), sx, wq, sw, b))


ACROSS = [(300, 1024, 512), (2048, 512, 1024), (40, 100, 60), (64, 7, 64), (33, 333, 1000), (20, 64, 64), (20, 65, 64),
          (152, 7248, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,F", ACROSS)
def test_several_transposed_operands(cuda, M, D, F):
    g = gen(M + D, cuda)
    dh, x, wg, wu, gate, up = case = gated_bwd_case(g, M, D, F)
    for a in (x, across(x)):
        gated_check(x, wg, wu, "silu", ops.gated_linear(a, across(wg), across(wu), "silu", save=True), True)
    gated_bwd_check(*case, "silu", ops.gated_linear_bwd(*(across(t) for t in case), "silu"))
    xq, sx, wq, sw, b = i8_case(g, M, F, D)
    i8_check(xq, sx, wq, sw, b, "none", ops.linear_i8(across(xq), sx, across(wq), sw, b))
    # captured: the copies belong to the graph
    xa, wa, qa = across(x), across(wg), across(xq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = ops.gated_linear(xa, wa, across(wu), "silu")
        y = ops.linear_i8(qa, sx, across(wq), sw, b)
    for seed in range(3):
        xa.copy_(randn(gen(seed, cuda), M, D))
        graph.replay()
        gated_check(xa, wg, wu, "silu", h, False)
        i8_check(xq, sx, wq, sw, b, "none", y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_kl_of_long_rows_captured(cuda, dtype):
    """Rows in chunks, two launches and a workspace: two graphs replayed in turn, with eager calls between; no entries."""
    sets = [distill_case(gen(s, cuda), 3, n, 9, dtype) for s, n in ((1, 70001), (2, 140000))]
    for s in sets:
        ops.distill_kl(*s)
    torch.cuda.synchronize()
    graphs, out = [torch.cuda.CUDAGraph() for _ in sets], []
    for graph, s in zip(graphs, sets):
        with torch.cuda.graph(graph):
            out.append(ops.distill_kl(*s, temperature=2.0))
    for rep in range(3):
        for s in sets:
            s[0].copy_(randn(gen(50 + rep, cuda), *s[0].shape, std=2.0, dtype=dtype))
        for graph in (*graphs, *graphs):
            graph.replay()
        for s, (dz, loss) in zip(sets, out):
            now = ops.distill_kl(*s, temperature=2.0)
            assert torch.equal(dz, now[0]) and torch.equal(loss, now[1])
            distill_check(*s, 2.0, 1.0, dz, loss)
    dz, loss = ops.distill_kl(sets[0][0], sets[0][1][:, :0], sets[0][2][:, :0])
    assert not dz.any() and not loss.any()


# ---------------------------------------------------------------------------------------------------------------
# whole numbers: sums of -1, 0 and 1 are exact in 32 bits in any order, so that one lost or doubled product shows
# ---------------------------------------------------------------------------------------------------------------
def signs(g, *shape):
    return torch.randint(-1, 2, shape, device=g.device, generator=g).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,F", [(1, 4099, 64), (1, 16384, 40), (2, 9000, 17), (16, 2055, 40), (17, 8192, 50), (20, 4104, 70),
                                   (32, 16385, 35), (33, 5001, 1), (65, 9000, 70), (90, 15608, 33), (128, 16383, 520),
                                   (152, 7248, 1024), (300, 4100, 129), (777, 1024, 2731), (1030, 2072, 2063),
                                   (4090, 72, 4090), (2075, 456, 4248), (1000, 8200, 1030), (1371, 8, 4804), (5970, 136, 645)])
def test_gated_linear_of_whole_numbers(cuda, M, D, F):
    g = gen(M + D + F, cuda)
    x, wg, wu = signs(g, M, D), signs(g, F, D), signs(g, F, D)
    G, U = (x.to(D64) @ w.to(D64).t() for w in (wg, wu))
    h, gate, up = ops.gated_linear(x, wg, wu, "none", save=True)
    assert torch.equal(gate, G.bfloat16()) and torch.equal(up, U.bfloat16())
    assert torch.equal(h, (G.float() * U.float()).bfloat16())  # (one fp32 product of exact factors, rounded once)


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,F", [*GATED_BWD, (71, 3392, 5760), (1, 4096, 8192), (16, 1024, 9000), (20000, 72, 40), (9000, 264, 520)])
def test_gated_linear_bwd_of_whole_numbers(cuda, M, D, F):
    g = gen(M + D + F, cuda)
    dh, gate, up = (signs(g, M, F) for _ in range(3))
    x, wg, wu = signs(g, M, D), signs(g, F, D), signs(g, F, D)
    dG, dU = (dh * up).to(D64), (dh * gate).to(D64)  # (-1, 0 and 1 again)
    dx, dwg, dwu = ops.gated_linear_bwd(dh, x, wg, wu, gate, up, "none")
    assert torch.equal(dx, (dG @ wg.to(D64) + dU @ wu.to(D64)).bfloat16())
    assert torch.equal(dwg, (dG.t() @ x.to(D64)).bfloat16()) and torch.equal(dwu, (dU.t() @ x.to(D64)).bfloat16())


# ---------------------------------------------------------------------------------------------------------------
# refusals (the arguments are looked at before the device: these run without a GPU)
# ---------------------------------------------------------------------------------------------------------------
def refused(match, f, *a, **k):
    with pytest.raises(RuntimeError, match=match):
        f(*a, **k)


def test_refusals():
    b, f = torch.bfloat16, torch.float32
    x, w, h = torch.zeros(4, 16, dtype=b), torch.zeros(8, 16, dtype=b), torch.zeros(4, 8, dtype=b)
    refused("unknown activation", ops.gated_linear, x, w, w, "swish")
    refused("x has dtype", ops.gated_linear, x.float(), w, w)
    refused("x must be a 2-D", ops.gated_linear, x[0], w, w)
    refused("w_gate has shape", ops.gated_linear, x, w[:, :8], w)
    refused("w_up has shape", ops.gated_linear, x, w, w[:4])
    refused("empty weights", ops.gated_linear, x, w[:0], w[:0])
    refused("on the GPU", ops.gated_linear, x, w, w)
    refused("unknown activation", ops.gated_linear_bwd, h, x, w, w, h, h, 3)
    refused("dh has shape", ops.gated_linear_bwd, h[:2], x, w, w, h, h)
    refused("gate has dtype", ops.gated_linear_bwd, h, x, w, w, h.float(), h)
    refused("up has shape", ops.gated_linear_bwd, h, x, w, w, h, h[:, :4])
    refused("on the GPU", ops.gated_linear_bwd, h, x, w, w, h, h)
    q, p = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(8, 16, dtype=torch.int8)
    s4, s8 = torch.zeros(4), torch.zeros(8)
    refused("x has dtype", ops.linear_i8, q.to(torch.uint8), s4, p, s8)
    refused("w has shape", ops.linear_i8, q, s4, p[:, :8], s8)
    refused("x_scale must be a vector of 4", ops.linear_i8, q, s8, p, s8)
    refused("w_scale has dtype", ops.linear_i8, q, s4, p, s8.double())
    refused("b must be a vector", ops.linear_i8, q, s4, p, s8, s4)
    refused("unknown activation", ops.linear_i8, q, s4, p, s8, None, "gelu")
    refused("out_dtype", ops.linear_i8, q, s4, p, s8, out_dtype=torch.float16)
    refused("131071", ops.linear_i8, torch.zeros(1, 131072, dtype=torch.int8), s4[:1],
            torch.zeros(1, 131072, dtype=torch.int8), s4[:1])
    refused("on the GPU", ops.linear_i8, q, s4, p, s8)
    refused("bf16 or fp32", ops.rmsnorm_i8, x.half(), x[0].half())
    refused("w must be a vector", ops.rmsnorm_i8, x, h[0])
    refused("w has dtype", ops.rmsnorm_i8, x, x[0].float())
    refused("residual has shape", ops.rmsnorm_i8, x, x[0], h)
    refused("eps", ops.rmsnorm_i8, x, x[0], eps=-1.0)
    refused("eps", ops.rmsnorm_i8, x, x[0], eps=float("nan"))
    refused("eps", ops.rmsnorm_i8, x, x[0], eps=float("inf"))
    refused("rows of 1 to 32768", ops.rmsnorm_i8, torch.zeros(1, 32769), torch.zeros(32769))
    refused("on the GPU", ops.rmsnorm_i8, x, x[0])
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    refused("bf16 or fp32", ops.distill_kl, x.half(), t, i)
    refused("t_index has dtype", ops.distill_kl, x, t, i.short())
    refused("t_index has shape", ops.distill_kl, x, t, i[:, :2])
    refused("t_logits has shape", ops.distill_kl, x, t[:2], i)
    refused("temperature", ops.distill_kl, x, t, i, temperature=0.0)
    refused("temperature", ops.distill_kl, x, t, i, temperature=float("inf"))
    refused("grad_dtype", ops.distill_kl, x.float(), t, i, grad_dtype=b)
    refused("at most 1024", ops.distill_kl, x, torch.zeros(4, 1025), torch.zeros(4, 1025, dtype=torch.int64))
    refused("no classes", ops.distill_kl, x[:, :0], t, i)
    refused("on the GPU", ops.distill_kl, x, t, i)


def test_native_refusals():
    """The launchers check by themselves: bad arguments raise before anything is launched."""
    K = ops.feedforward._K
    err = ops.feedforward._C.MccError
    for call in (lambda: K.gated_forward(33, 9, 8, 0, 0, 9, 0, 0, 9, 0, any=True), lambda: K.gated_forward(1, 9, 8, 0, 0, 9, 0, 0, -9, 0, any=True),
                 lambda: K.linear_i8(33, 1, 9, 0, 0, 9, 0, 0, 9, 0, 0, 0, False, any=True),
                 lambda: K.gated_forward(1, 8, 8, 9, 0, 8, 0, 0, 8, 0), lambda: K.gated_forward(1, 8, 8, 0, 0, 4, 0, 0, 8, 0),
                 lambda: K.gated_forward(1, 8, 8, 0, 2, 8, 0, 0, 8, 0), lambda: K.gated_forward(1, 0, 8, 0, 0, 8, 0, 0, 8, 0),
                 lambda: K.gated_backward(1, 8, 8, 0, 0, 0, 0, 0, 4, 0, 0, 8, 0, 0, 0),
                 lambda: K.linear_i8(1, 1, 131072, 0, 0, 131072, 0, 0, 131072, 0, 0, 0, False),
                 lambda: K.linear_i8(1, 1, 16, 3, 0, 16, 0, 0, 16, 0, 0, 0, False),
                 lambda: K.pad_rows([(0, 0, 8, 24, 1, 8)]), lambda: K.pad_rows([(0, 0, 8, 16, 1, 17)]),
                 lambda: K.pad_rows([(0, 8, 8, 16, 1, 8)]), lambda: K.pad_rows([(0, 0, 8, 16, 1, 0)]),
                 lambda: K.rmsnorm_i8(1, 40000, False, 0, 40000, 0, 0, 0, 0.0, 0, 0, 0),
                 lambda: K.distill_kl(1, 8, 2000, 0, 8, True, 0, True, 0, True, 1.0, 1.0, 0, True, 0, 0),
                 lambda: K.distill_kl(1, 8, 1, 0, 8, True, 0, True, 0, True, 0.0, 1.0, 0, True, 0, 0),
                 lambda: K.distill_kl(1, 200000, 1, 0, 200000, True, 0, True, 0, True, 1.0, 1.0, 0, True, 0, 0)):
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("M,D,F", [(4_000_001, 8, 8), (1, 8, (1 << 20) + 1), (0, 8, 8), (8, 0, 8), (8, 8, 0)])
def test_backward_sizes_are_refused_before_a_workspace_is_made(M, D, F):
    with pytest.raises(ops.feedforward._C.MccError, match="gated_linear_bwd: (too many rows|empty problem)"):
        ops.feedforward._K.gated_backward_bytes(M, D, F)


@pytest.mark.parametrize("M", [1, 32])
@pytest.mark.parametrize("K", [16, 8192])
def test_more_output_columns_than_a_grid_takes_are_refused(M, K):
    k, err = ops.feedforward._K, ops.feedforward._C.MccError
    with pytest.raises(err, match="linear_i8: too many output columns"):
        k.linear_i8(M, 1 << 30, K, 0, 0, K, 0, 0, K, 0, 0, 0, False)
    with pytest.raises(err, match="gated_linear: too many output columns"):
        k.gated_forward(M, K, 1 << 30, 0, 0, K, 0, 0, K, 0)


def test_rows_longer_than_a_buffer_offset_takes_are_refused():
    k, err = ops.feedforward._K, ops.feedforward._C.MccError
    for M in (1, 33):
        with pytest.raises(err, match="gated_linear: row pitch too large"):
            k.gated_forward(M, 1 << 22, 8, 0, 0, 1 << 22, 0, 0, 1 << 22, 0)
