"""Feed-forward, 8-bit and distillation operators of ``ops`` on the MI355X.

Every output is compared element by element with the definition in 64 bits.
The bounds are worst cases of the arithmetic that the kernels document:

  * a sum of K products in 32 bits: each of the K additions is off by at most
    2^-23 of the partial sum (a matrix unit may truncate), so by at most
    K 2^-23 sum_k |a_k b_k| in all;
  * a rounding to bf16 is off by at most 2^-8 of the value, to fp32 2^-24;
  * an activation in 32 bits by a few units in the last place (2^-20 allowed).
"""

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
         (1000, 520, 130), (4097, 64, 1030), (2050, 136, 4232)]


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
      (128, 128, 640), (130, 70, 130), (640, 1000, 512), (1030, 4100, 176), (4100, 4360, 144), (70, 17, 20000)]


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
