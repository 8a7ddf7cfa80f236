"""Plain 64-bit forms of the 8-bit integer operators, and how far a correct result may be from them.

Bounds.  The integer sum is exact.  With u = 2^-24 (half a step of float32), the device forms fl(fl(acc) sw) sa + bias, the last
two steps fused: two roundings of the product and one of the sum, so a float32 result is within 3 u (|p| + |bias|) of
p + bias, p = acc sa sw; the bound is 2^-22 (|p| + |bias|).  The residual form adds resid + alpha (...) in one fused step: |alpha| times it, and u of
the result.  A bf16 output is rounded once more, half a step = 2^-8 of the value.  Swish and the GLU gate use the hardware's
exponential and reciprocal: the exponential's argument x log2(e) is rounded (|x| 2^-24 relative error of the result), each
instruction is good to about a step; for the |x| <= 90 of these tests that is below 2^-16 of the value.  Swish's slope is
at most 1.1, the sigmoid's 1 / 4."""

import math

import torch


def quantize64(x: torch.Tensor):
    """(codes, scale) of float rows from the definition in 64 bits; the scale rounded to float32 as it is stored."""
    x = x.to(torch.float64)
    amax = x.abs().amax(dim=-1, keepdim=True)
    top = torch.where(amax > 0, amax, torch.full_like(amax, 127.0))
    return (127.0 * x / top).round(), (top / 127.0).squeeze(-1)


def product64(codes_a, scale_a, codes_w, scale_w):
    return (codes_a.double() @ codes_w.double().t()) * scale_a.double()[:, None] * scale_w.double()[None, :]


def finish64(p, bias, epilogue, resid=None, alpha=1.0):
    """(result, bound) of an epilogue on the exact products p [m, n]."""
    b = torch.zeros_like(p[0]) if bias is None else bias.double()
    y, err = p + b, 2.0 ** -22 * (p.abs() + b.abs())
    if epilogue == "float":
        return y, err
    if epilogue == "residual":
        r = resid.double() + alpha * y
        return r, abs(alpha) * err + 2.0 ** -23 * r.abs()
    if epilogue == "swish":
        y, err = y * torch.sigmoid(y), 1.1 * err
    elif epilogue == "glu":
        t, e = y.view(y.shape[0], -1, 2, 16), err.view(y.shape[0], -1, 2, 16)
        sig = torch.sigmoid(t[:, :, 1])
        y, err = t[:, :, 0] * sig, e[:, :, 0] + 0.25 * t[:, :, 0].abs() * e[:, :, 1]
        y, err = y.reshape(p.shape[0], -1), err.reshape(p.shape[0], -1)
    return y, err + y.abs() * (2.0 ** -8 + 2.0 ** -16) + 1e-37


def assert_within(got, want, bound):
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = torch.where(nan, torch.zeros_like(want), (got - want).abs() - bound)
    assert float(off.max()) <= 0, (float(off.max()), int((off > 0).sum()), off.argmax())


def weight_codes(n, k, gen):
    codes = (torch.randn((n, k), generator=gen) * 40).round().clamp(-128, 127).to(torch.int8)
    scale = (0.5 + torch.rand((n,), generator=gen)) / (40 * math.sqrt(k))
    return codes, scale
