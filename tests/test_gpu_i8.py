"""GPU tests of the 8-bit integer operators: codes and scales against the definition (bit for bit), products and epilogues
against 64-bit sums of the same codes within bounds that tests/i8_tools.py derives, and the calls around them (strides,
empty batches, aliasing, streams, graphs, offsets past 32 bits).  Parity unpinned against the reference, which has none."""

import math

import pytest
import torch

from omnilingual_asr import _hip as H
from omnilingual_asr import ops
from omnilingual_asr.weights import quantize_rows_i8
from tests.i8_tools import assert_within, finish64, product64, quantize64, weight_codes

pytestmark = pytest.mark.gpu


def _quant(x, ldy=None, fill=77):
    rows, k = x.shape
    kp = (k + 63) // 64 * 64
    y = torch.full((rows, ldy or kp), fill, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), -1.0, device="cuda")
    H.check(H.lib().oasr_quant_i8_rows(x.data_ptr(), x.stride(0), rows, k, y.data_ptr(), y.shape[1], s.data_ptr(), H.current_stream_ptr()))
    torch.cuda.synchronize()
    return y, s


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 63), (5, 64), (7, 65), (4, 511), (9, 512), (6, 1000), (33, 1024), (5, 2047),
                                    (17, 4096), (3, 8191), (5, 16384), (2, 16385), (3, 40001),
                                    (9000, 100), (9000, 1030), (9001, 4090), (8200, 4100), (700, 8192)])
def test_quant_rows_bit_for_bit(rows, k):
    g = torch.Generator().manual_seed(rows * 7 + k)
    x = (torch.randn((rows, k), generator=g) * torch.rand((rows, 1), generator=g) * 4).to(torch.bfloat16)
    x[rows // 2] = x[rows // 2].abs().max() * torch.tensor([1.0, 0.5, -0.5, 0.25]).repeat(k // 4 + 1)[:k]   # ties: 63.5, 31.75
    if rows > 2:
        x[0] = 0
    pitch = k + 3                                       # rows that start at any alignment
    buf = torch.zeros((rows, pitch), dtype=torch.bfloat16, device="cuda")
    buf[:, :k] = x.cuda()
    kp = (k + 63) // 64 * 64
    y, s = _quant(buf[:, :k], ldy=kp + 16)
    want, scale = quantize64(x)
    assert torch.equal(y[:, :k].cpu().double(), want)
    assert (y[:, k:kp] == 0).all() and (y[:, kp:] == 77).all()
    assert torch.equal(s.cpu(), (x.float().abs().amax(1) / 127.0).masked_fill(x.abs().amax(1) == 0, 1.0))


def test_quant_rows_at_the_ends_of_the_range():
    """Smallest and largest rows keep their codes; NaN and infinity show in the scale, whatever else the row holds."""
    x = torch.zeros((8, 70), dtype=torch.bfloat16)
    x[0, :3] = torch.tensor([9.2e-41, -9.2e-41, 0.0])                   # the smallest bf16
    x[1, :3] = torch.tensor([3.3895e38, -1.69e38, 1e30])                # the largest
    x[2, :3] = torch.tensor([1e-38, 5e-39, -2.5e-39])
    x[3, :3] = torch.tensor([float("nan"), 1.0, 2.0])
    x[4, :3] = torch.tensor([float("inf"), 1.0, -2.0])
    x[5, :3] = torch.tensor([-float("inf"), float("nan"), -2.0])
    x[6, 69] = -5.0
    y, s = _quant(x.cuda())
    want, _ = quantize64(x[[0, 1, 2, 6, 7]])
    assert torch.equal(y[[0, 1, 2, 6, 7], :70].cpu().double(), want)
    sc = s.cpu()
    assert torch.isnan(sc[3]) and torch.isinf(sc[4]) and torch.isnan(sc[5]) and sc[7] == 1.0
    assert torch.allclose(sc[[0, 1, 2, 6]].double(), x[[0, 1, 2, 6]].double().abs().amax(1) / 127, rtol=1e-2, atol=0)
    codes, scale = weight_codes(33, 70, torch.Generator().manual_seed(1))
    out = ops.LinearI8.from_codes(codes.cuda(), scale.cuda())(x.cuda(), epilogue="float").cpu()
    assert torch.isnan(out[3:6]).all() and torch.isfinite(out[[0, 1, 2, 6, 7]]).all()


SHAPES = [(1, 1, 1), (1, 33, 64), (1, 1024, 512), (2, 1000, 1000), (3, 64, 65), (15, 96, 63), (16, 128, 128), (17, 130, 640),
          (33, 4096, 256), (64, 512, 4096), (99, 2048, 1024), (127, 257, 191), (128, 128, 64), (129, 384, 320), (200, 777, 1000),
          (256, 256, 64), (300, 96, 16448), (513, 1024, 512), (1000, 4096, 64), (1504, 1024, 1024), (2100, 640, 192),
          (4096, 512, 512), (8200, 1056, 320), (2100, 4128, 128), (4500, 2080, 64), (2049, 4097, 65),
          (48, 1000, 8192), (300, 2048, 4096), (400, 700, 4096), (1504, 1024, 4096), (1500, 1000, 4100), (2000, 2100, 4096), (64, 16400, 100),
          (17, 500, 500), (40, 70, 1024), (256, 1000, 1000), (33, 4000, 960), (16, 2000, 1024), (15, 300, 1090), (5, 64, 3210), (3, 96, 16384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("epilogue", ["bias", "swish", "glu", "residual", "float"])
def test_linear_i8(m, n, k, epilogue):
    g = torch.Generator().manual_seed(m + 3 * n + 7 * k)
    if epilogue == "glu":
        n = (n + 31) // 32 * 32
    x = (torch.randn((m, k), generator=g) * (0.2 + 2 * torch.rand((m, 1), generator=g))).to(torch.bfloat16)
    codes, scale = weight_codes(n, k, g)
    bias = torch.randn((n,), generator=g) if n % 5 else None
    resid = torch.randn((m, n), generator=g) if epilogue == "residual" else None
    layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), None if bias is None else bias.cuda())
    got = layer(x.cuda(), epilogue=epilogue, resid=None if resid is None else resid.cuda(), alpha=0.5)
    qa, _ = quantize64(x)
    sa = (x.float().abs().amax(1) / 127.0).masked_fill(x.abs().amax(1) == 0, 1.0)
    p = product64(qa.cuda(), sa.cuda(), codes.cuda(), scale.cuda()).cpu()
    assert_within(got, *finish64(p, bias, epilogue, resid, 0.5))


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("epilogue", ["bias", "swish", "glu", "residual", "float"])
def test_epilogues_up_to_the_ends_of_float32(m, epilogue):
    """Pre-activations as large as the type goes: a finite one gives a finite result, saturated gates are 0 and 1."""
    g = torch.Generator().manual_seed(m)
    ends = torch.tensor([3.3e38, 2.4e38, 1e38, 1e30, 1e4, 100.0, 89.0, 3.0])
    bias = torch.cat([ends, -ends, torch.zeros(16)]).repeat(2)
    bias[48:] = torch.cat([ends, -ends])                     # the second group's gates
    bias[32:48] = torch.cat([-ends, ends]) * 0.5
    codes, scale = weight_codes(64, 70, g)
    x = torch.zeros((m, 70), dtype=torch.bfloat16)
    x[0] = torch.randn(70, generator=g).to(torch.bfloat16)
    resid = torch.randn((m, 64), generator=g) if epilogue == "residual" else None
    layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), bias.cuda())
    got = layer(x.cuda(), epilogue=epilogue, resid=None if resid is None else resid.cuda(), alpha=0.5)
    qa, _ = quantize64(x)
    sa = (x.float().abs().amax(1) / 127.0).masked_fill(x.abs().amax(1) == 0, 1.0)
    assert torch.isfinite(got).all()
    assert_within(got, *finish64(product64(qa, sa, codes, scale), bias, epilogue, resid, 0.5))


def _norm64(x, w, b, swish=0):
    """LayerNorm (and Swish) in 64 bits, and how far a float32 evaluation may be.  With u = 2^-24: the mean is a tree of at
    most 24 additions deep, so it is within 24 u mean|x|, and mean|x| rstd <= sqrt(1 + mean^2 / var), below 1.1 for
    these rows; rstd is good to 15 u; the affine map adds three roundings: |dv| <= |g| (27 u + 15 u |xhat|) + 3 u (|v| + |h|),
    which is below 2^-19 (|g| + |g xhat| + |h|).  Swish: slope at most 1.1, and 2^-16 of the value (tests/i8_tools.py)."""
    x, w, b = x.double(), w.double(), b.double()
    hat = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
    v, off = hat * w + b, 2.0 ** -19 * (w.abs() + (hat * w).abs() + b.abs())
    return (v * torch.sigmoid(v), 1.1 * off + 2.0 ** -16 * v.abs()) if swish else (v, off)


@pytest.mark.parametrize("m,n,k", [(8200, 4128, 2112), (3000, 16416, 1050), (20000, 2080, 1024), (6016, 4096, 4096)])
@pytest.mark.parametrize("epilogue", ["bias", "swish", "glu", "residual", "float"])
def test_linear_i8_large(m, n, k, epilogue):
    """Sizes that take the 256 x 256 form (by row bands and by flat tile ranges), ragged on every side; compared on the device."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16)
    codes = (torch.randn((n, k), generator=g, device="cuda") * 40).round().clamp(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand((n,), generator=g, device="cuda")) / (40 * math.sqrt(k))
    bias = torch.randn((n,), generator=g, device="cuda")
    resid = torch.randn((m, n), generator=g, device="cuda") if epilogue == "residual" else None
    got = ops.LinearI8.from_codes(codes, scale, bias)(x, epilogue=epilogue, resid=resid, alpha=0.5)
    qa, _ = quantize64(x)
    want, bound = finish64(product64(qa, x.float().abs().amax(1) / 127.0, codes, scale), bias, epilogue, resid, 0.5)
    assert float(((got.double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("rows,d,swish", [(9, 512, 0), (130, 1024, 0), (6, 4096, 1), (5, 2048, 1), (3, 256, 0), (1, 1024, 0)])
def test_layernorm_i8(rows, d, swish):
    """Scales and codes against the 64-bit rows: a scale within the rows' bound / 127 (and its own rounding), a code within
    half a step of 127 v / max|v|, plus what the bound on v is worth in steps, plus 2^-16 for the kernel's two roundings of the
    quotient (127 * 2^-23)."""
    g = torch.Generator().manual_seed(rows + d)
    x = (torch.randn((rows, d), generator=g) * 3 + 0.5).cuda()
    if rows > 1:
        x[1] = 0.25                                   # a constant row: normalises to the bias, exactly
    w1, b1, w2, b2 = (torch.randn((d,), generator=g).cuda() for _ in range(4))
    L, st = H.lib(), H.current_stream_ptr()
    xa = x.clone()
    q = torch.full((rows, d), 99, dtype=torch.int8, device="cuda")
    s = torch.zeros((rows,), device="cuda")

    def check(v, off):
        top = s.double()[:, None] * 127
        assert ((top[:, 0] - v.abs().amax(1)).abs() <= off.amax(1) + 2.0 ** -22 * top[:, 0]).all()
        assert ((q.double() - 127 * v / top).abs() <= 0.5 + 127 * off / top + 2.0 ** -16).all()
        assert int(q.abs().max()) == 127

    H.check(L.oasr_layernorm_i8(xa.data_ptr(), w1.data_ptr(), b1.data_ptr(), q.data_ptr(), s.data_ptr(), rows, d, 1e-5, swish, st))
    torch.cuda.synchronize()
    assert torch.equal(xa, x)
    check(*_norm64(x, w1, b1, swish))
    if not swish:
        H.check(L.oasr_layernorm2_i8(xa.data_ptr(), w1.data_ptr(), b1.data_ptr(), w2.data_ptr(), b2.data_ptr(), q.data_ptr(),
                                     s.data_ptr(), rows, d, 1e-5, st))
        torch.cuda.synchronize()
        v, off = _norm64(x, w1, b1)
        assert ((xa.double() - v).abs() <= off).all()
        check(*_norm64(xa, w2, b2))


@pytest.mark.parametrize("m,k,epilogue", [(1, 512, "bias"), (77, 1024, "swish"), (301, 2048, "residual")])
def test_normed_linear(m, k, epilogue):
    """LayerNorm in 64 bits against the call: a row's normalised values differ by float32 roundings, so a code may fall on
    the other side of a tie; the chance per value is about 2^-23 * 127 * a few, so at most a handful of the row's k codes do
    (allowed: 4), each moving an output by one step of x times one weight."""
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn((m, k), generator=g) * 2 + 0.3
    gain, shift = 1 + 0.2 * torch.randn((k,), generator=g), 0.2 * torch.randn((k,), generator=g)
    codes, scale = weight_codes(96, k, g)
    bias = torch.randn((96,), generator=g)
    resid = torch.randn((m, 96), generator=g) if epilogue == "residual" else None
    layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), bias.cuda())
    got = layer.normed(x.cuda(), gain.cuda(), shift.cuda(), epilogue=epilogue, alpha=2.0,
                       resid=None if resid is None else resid.cuda())
    x64 = x.double()
    y = (x64 - x64.mean(1, keepdim=True)) / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + 1e-5) * gain.double() + shift.double()
    qa, sa = quantize64(y)
    p = product64(qa, sa, codes, scale)
    want, bound = finish64(p, bias, epilogue, resid, 2.0)
    step = 4 * sa[:, None] * 128 * scale.double()[None, :] + 2.0 ** -20 * p.abs()      # and the float32 scale of the row
    assert_within(got, want, bound + 2.2 * step)


def test_quantised_weight_constructor_and_leading_dimensions():
    g = torch.Generator().manual_seed(5)
    w, x = torch.randn((40, 96), generator=g) / 10, torch.randn((2, 3, 96), generator=g).to(torch.bfloat16)
    layer = ops.LinearI8(w.cuda())
    codes, scale = quantize_rows_i8(w)
    got = layer(x.cuda(), epilogue="float")
    assert got.shape == (2, 3, 40) and torch.equal(layer.scale.cpu(), scale)
    assert torch.equal(got, ops.LinearI8.from_codes(codes.cuda(), scale.cuda())(x.cuda(), epilogue="float"))
    assert torch.equal(layer(x[0, 0].cuda(), epilogue="float"), got[0, 0])
    assert layer(x[:0].cuda()).shape == (0, 3, 40) and layer(x.cuda()[:, :0]).shape == (2, 0, 40)
    # the quantised layer is close to the float one: two quantisations, each within half a step of its row's maximum
    exact = x.double() @ w.double().t()
    bound = 96 * (x.double().abs().amax(-1, keepdim=True) * w.double().abs().amax(1)) * (1 / 127)
    assert ((got.double().cpu() - exact).abs() <= bound).all()


def test_strided_rows_in_and_out_and_untouched_surroundings():
    g = torch.Generator().manual_seed(6)
    for n, k, pad in ((70, 100, 5), (96, 128, 32), (33, 65, 1)):
        m = 37
        codes, scale = weight_codes(n, k, g)
        layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), torch.randn((n,), generator=g).cuda())
        x = torch.randn((m, k + pad), generator=g).to(torch.bfloat16).cuda()
        dense = layer(x[:, :k].contiguous())
        assert torch.equal(layer(x[:, :k]), dense)
        for dtype, epi in ((torch.bfloat16, "bias"), (torch.float32, "float"), (torch.float32, "residual")):
            buf = torch.full((m + 2, n + pad), 7.0, dtype=dtype, device="cuda")
            view = buf[1:-1, :n]
            want = layer(x[:, :k], epilogue=epi, resid=torch.full((m, n), 7.0, device="cuda") if epi == "residual" else None)
            layer(x[:, :k], epilogue=epi, resid=view if epi == "residual" else None, out=view)
            assert torch.equal(view, want)
            if epi == "residual":        # a residual with a pitch of its own
                assert torch.equal(layer(x[:, :k], epilogue=epi, resid=torch.full((m, n + 3), 7.0, device="cuda")[:, :n]), want)
            assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, n:] == 7).all()
        # codes with a pitch of their own
        wide = torch.full((n, k + pad), 55, dtype=torch.int8, device="cuda")
        wide[:, :k] = codes.cuda()
        assert torch.equal(ops.LinearI8.from_codes(wide[:, :k], scale.cuda(), layer.bias)(x[:, :k]), dense)


def test_every_row_is_its_own_whatever_the_batch():
    """A token's result does not depend on the rows around it, nor on which kernel its batch size selects: bit for bit."""
    g = torch.Generator().manual_seed(8)
    for n, k in ((512, 1024), (777, 1000), (1024, 4096)):
        codes, scale = weight_codes(n, k, g)
        layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), torch.randn((n,), generator=g).cuda())
        x = torch.randn((3000, k), generator=g).to(torch.bfloat16).cuda()
        for epi in ("bias", "swish", "float"):
            full = layer(x, epilogue=epi)
            for m in (1, 2, 7, 16, 31, 64, 100, 129, 300, 513, 1500):
                assert torch.equal(layer(x[1000: 1000 + m], epilogue=epi), full[1000: 1000 + m]), (n, k, epi, m)


def test_largest_sums_are_exact():
    """k = 131072 with codes -128 and 127 alternating in sign: the sums reach 2^31 - 2^24 and come back exact to float32."""
    k = 131072
    x = torch.ones((3, k), dtype=torch.bfloat16, device="cuda")
    x[1] = -1
    codes = torch.full((32, k), -128, dtype=torch.int8, device="cuda")
    codes[1] = 127
    layer = ops.LinearI8.from_codes(codes, torch.ones((32,), device="cuda"))
    got = layer(x, epilogue="float").double().cpu()
    assert (got[0, 0], got[1, 0]) == (-128.0 * k, 128.0 * k)
    assert abs(got[0, 1] - 127.0 * k) <= 2 ** -22 * 127 * k
    with pytest.raises(ValueError, match="131072"):
        ops.LinearI8.from_codes(torch.zeros((1, k + 1), dtype=torch.int8, device="cuda"), torch.ones((1,), device="cuda"))


def test_parameters_of_a_module():
    """Weights and biases that a module holds (they require gradients) make a layer that keeps no graph of them."""
    lin = torch.nn.Linear(96, 40, device="cuda")
    layer = ops.LinearI8(lin.weight, lin.bias)
    x = torch.randn((7, 96), device="cuda").to(torch.bfloat16)
    assert not layer.scale.requires_grad
    assert torch.equal(layer(x), ops.LinearI8(lin.weight.detach().clone(), lin.bias.detach().clone())(x))


def test_offsets_past_32_bits():
    m, n, k = 66000, 33000, 64
    g = torch.Generator().manual_seed(9)
    codes, scale = weight_codes(n, k, g)
    layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda())
    x = torch.randn((m, k), generator=g).to(torch.bfloat16).cuda()
    out = layer(x)
    assert out.numel() > 1 << 31
    for lo in (0, 40000, m - 300):
        assert torch.equal(out[lo: lo + 300], layer(x[lo: lo + 300]))
    del out
    far = torch.zeros(((1 << 26) * 40,), dtype=torch.bfloat16, device="cuda").view(40, 1 << 26)[:, :k]
    far.copy_(x[:40])
    assert torch.equal(layer(far), layer(x[:40]))


def test_refusals_on_the_device():
    g = torch.Generator().manual_seed(10)
    codes, scale = weight_codes(48, 64, g)
    c, s = codes.cuda(), scale.cuda()
    layer = ops.LinearI8.from_codes(c, s)
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    y = x.clone()
    z = torch.zeros((5, 48), device="cuda")
    wide, f, v = ops.LinearI8(torch.ones((16, 512), device="cuda")), torch.zeros((4, 512), device="cuda"), torch.ones(520, device="cuda")
    bad = [
        (lambda: layer(x[:, :63]), "64 columns"), (lambda: layer(x.float()), "bfloat16"), (lambda: layer(x, epilogue="gelu"), "epilogue"),
        (lambda: layer(x, epilogue="glu"), "multiple of 32"), (lambda: layer(x, epilogue="residual"), "resid"),
        (lambda: layer(x, resid=torch.zeros((4, 48), device="cuda")), "resid"),
        (lambda: layer(x, epilogue="residual", resid=torch.zeros((4, 47), device="cuda")), "resid"),
        (lambda: layer(x, out=torch.zeros((4, 47), dtype=torch.bfloat16, device="cuda")), "shape"),
        (lambda: layer(x, out=torch.zeros((4, 48), device="cuda")), "bfloat16"),
        (lambda: layer(x, out=torch.zeros((48, 4), dtype=torch.bfloat16, device="cuda").t()), "contiguous rows"),
        (lambda: layer(y, out=y[:, :48]), "overlap x"),
        (lambda: layer(x, epilogue="residual", resid=z[:4], out=z[1:]), "resid may be out"),
        (lambda: layer(x.t()[:, :1].expand(64, 64)[:4]), "contiguous rows"),
        (lambda: layer(torch.zeros((1, 64), dtype=torch.bfloat16, device="cuda").expand(4, 64)), "overlap"),
        (lambda: layer.normed(x.float(), s, s), "normed"), (lambda: layer.normed(x, s, s), "float32"),
        (lambda: layer(x, out=[0.0]), "out must be"), (lambda: layer(x, epilogue="residual", resid=1.0), "resid"),
        (lambda: wide.normed(f, v[:512], v[1:513]), "aligned"), (lambda: wide.normed(f, v[:512], None), "given"),
        (lambda: ops.LinearI8.from_codes(c, 1.0), "scale"),
        (lambda: ops.LinearI8.from_codes(c, s[:4]), "scale"), (lambda: ops.LinearI8.from_codes(c, None), "scale"),
        (lambda: ops.LinearI8.from_codes(c, s, s.double()), "bias"), (lambda: ops.LinearI8.from_codes(c.t(), s), "contiguous rows"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()


def test_streams_and_repeated_graph_replays():
    """Captured calls on one layer, replayed between eager calls of the same layer on another stream: each equals its eager
    result (the workspaces belong to the calls)."""
    g = torch.Generator().manual_seed(11)
    codes, scale = weight_codes(512, 1024, g)
    layer = ops.LinearI8.from_codes(codes.cuda(), scale.cuda(), torch.randn((512,), generator=g).cuda())
    gain, shift = torch.ones((1024,), device="cuda"), torch.zeros((1024,), device="cuda")
    for m in (1, 60, 700):
        x = torch.randn((m, 1024), generator=g).to(torch.bfloat16).cuda()
        other = torch.randn((m, 1024), generator=g).to(torch.bfloat16).cuda()
        resid = torch.randn((m, 512), generator=g).cuda()
        call = lambda t: (layer(t), layer(t, epilogue="residual", resid=resid), layer.normed(t.float(), gain, shift))  # noqa: E731
        side = torch.cuda.Stream()
        want_x, want_other = call(x), call(other)
        torch.cuda.synchronize()
        buf = x.clone()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = call(buf)
            graphs.append((graph, out))
        for rep in range(4):
            src, want = ((x, want_x), (other, want_other))[rep & 1]
            buf.copy_(src)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                eager = call(other)
            for graph, out in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for graph, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert all(torch.equal(a, b) for a, b in zip(eager, want_other))


def test_encoder_int8_against_the_quantising_oracle():
    """GTINY (2 blocks), ragged batch, every large projection in 8-bit integers.  What to expect, by arithmetic: rounding to a
    step max / 127 leaves an rms error of max / (127 sqrt 12); activations reach about 3.7 of their rms (max over 512), the
    uniform weights sqrt 3: relative errors 0.0084 and 0.0039 per operand, 0.0093 per product, against e4m3's 0.026 per
    operand and 0.037 per product, whose two blocks end 3.6e-2 from the float32 oracle: int8 should end near 0.9e-2 (bound
    2e-2).  Two correct implementations end at up to about two thirds of that from one another after two blocks, since values next
    to a rounding step fall on either side (bound 1.3e-2)."""
    from omnilingual_asr.engine_hip import HipEngine
    from omnilingual_asr.weights import GEOMETRIES, init_random_weights
    from oracle import conformer as OC
    from oracle import logmel as OL
    from tests.test_gpu_ops import synth_pcm

    g = GEOMETRIES["GTINY"]
    og = OC.Geometry(name=g.name, d_model=g.d_model, ffn_dim=g.ffn_dim, n_heads=g.n_heads, n_layers=g.n_layers)
    w = init_random_weights(g, 21)
    pcm = synth_pcm(2, 64000, seed=5)
    n_valid = [64000, 41000]
    feats, lens = OL.features_batch(pcm.numpy(), n_valid)
    enc_w = {k: v for k, v in w.items() if not k.startswith("ctc_")}
    ft, lt = torch.from_numpy(feats), torch.from_numpy(lens)
    emulated = OC.forward(ft, lt, enc_w, og, int8=True, device_rounding=True)
    plain = OC.forward(ft, lt, enc_w, og)
    h8, l8 = HipEngine("GTINY", weights=w, int8=True).encode_batch(pcm, n_valid)
    h16 = HipEngine("GTINY", weights=w).encode_batch(pcm, n_valid)[0].cpu()
    h8 = h8.cpu()
    rel = lambda a, b: float((a - b).norm() / b.norm())  # noqa: E731
    for i, n in enumerate(lens):
        assert int(l8[i]) == int(n)
        print("int8 against emulation %.2e, float32 %.2e" % (rel(h8[i, :n], emulated[i, :n]), rel(h8[i, :n], plain[i, :n])))
        assert rel(h8[i, :n], emulated[i, :n]) <= 1.3e-2
        assert rel(h8[i, :n], plain[i, :n]) <= 2e-2
        assert rel(h8[i, :n], h16[i, :n]) > 2e-3              # and not the bf16 path
    assert torch.isfinite(h8).all()
    with pytest.raises(ValueError, match="exclude"):
        HipEngine("GTINY", weights=w, int8=True, fp8=True)


def test_encoder_int8_unfused_convolution_width():
    """One block at d = 4096 (LayerNorm + Swish of the convolution branch goes straight to int8 rows there)."""
    import dataclasses
    from omnilingual_asr.engine_hip import HipEngine
    from omnilingual_asr.weights import GEOMETRIES, init_random_weights
    from oracle import conformer as OC
    from oracle import logmel as OL
    from tests.test_gpu_ops import synth_pcm

    g = dataclasses.replace(GEOMETRIES["G7B"], n_layers=1, ffn_dim=2048)
    og = OC.Geometry(name=g.name, d_model=g.d_model, ffn_dim=g.ffn_dim, n_heads=g.n_heads, n_layers=1)
    w = init_random_weights(g, 31)
    pcm = synth_pcm(1, 32000, seed=6)
    feats, lens = OL.features_batch(pcm.numpy(), [32000])
    enc_w = {k: v for k, v in w.items() if not k.startswith("ctc_")}
    ft, lt = torch.from_numpy(feats), torch.from_numpy(lens)
    n = int(lens[0])
    want = OC.forward(ft, lt, enc_w, og, int8=True, device_rounding=True)[0, :n]
    got = HipEngine(g, weights=w, int8=True).encode_batch(pcm, [32000])[0][0, :n].cpu()
    assert float((got - want).norm() / want.norm()) <= 1.3e-2


def test_int8_transcription_with_scores():
    """The whole run as a user makes it: int8 encoder, greedy decode, scores of what was decoded, against 64-bit scores of the
    engine's own logits; a second batch of the same shape gets its own."""
    from omnilingual_asr.engine_hip import HipEngine
    from omnilingual_asr.weights import CTC_LOGIT_PITCH
    from tests.test_gpu_ops import synth_pcm
    from tests.test_gpu_token_scores import close, reference

    eng = HipEngine("GTINY", seed=4, int8=True)
    for seed in (1, 2):
        pcm = synth_pcm(3, 48000, seed=seed)
        hidden, lengths, toks = eng.transcribe_batch(pcm, [48000, 20000, 0])
        hidden2, lengths2, toks2, scores = eng.transcribe_batch(pcm, [48000, 20000, 0], alternatives=3)
        assert len(scores) == 3 and sum(len(t[0]) for t in toks) > 0
        t_pad = hidden.shape[1]
        logits = eng._buffers[(3, t_pad)]["logits"][: 3 * t_pad].view(3, t_pad, CTC_LOGIT_PITCH)[:, :, : eng.geometry.vocab_size].cpu()
        for b in range(3):
            ids, frames = toks2[b]
            assert (ids == toks[b][0]).all() and (frames == toks[b][1]).all()
            s = scores[b]
            assert s.logprobs.shape == s.entropy.shape == (len(ids),) and s.ids.shape == s.best.shape == (len(ids), 3)
            if not len(ids):
                continue
            lp, ent, top, best = reference(logits[b, frames], torch.from_numpy(ids)[:, None], 3)
            close(torch.from_numpy(s.logprobs)[:, None], lp, lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
            close(torch.from_numpy(s.entropy), ent, lambda w: 2.0 ** -16 * (1 + w))
            close(torch.from_numpy(s.best), best, lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
            assert (s.ids == top.numpy()).all() and (s.ids[:, 0] == ids).all()
    with pytest.raises(ValueError, match="decode"):
        eng.score(torch.zeros((5, 7), dtype=torch.int32, device="cuda"), torch.zeros((5, 7), dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("m,n,k", [(100, 4096, 4160), (50, 8192, 1088), (300, 4100, 2050), (900, 1024, 2048), (1000, 1000, 1100), (130, 1030, 1030),
                                   (800, 3000, 700), (2500, 1000, 500), (1037, 2081, 1025)])
def test_every_tile_is_computed_once(m, n, k):
    """Tiles dealt to the chip's parts as blocks, ragged ones among them: every output is there and exact."""
    g = torch.Generator().manual_seed(m + n + k)
    a = torch.randint(-3, 4, (m, k), generator=g).to(torch.bfloat16)
    a[:, 0] = 127                                       # every row's scale is 1, its codes are its values
    codes = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    layer = ops.LinearI8.from_codes(codes.cuda(), torch.ones((n,), device="cuda"))
    out = torch.full((m, n), float("nan"), device="cuda")
    layer(a.cuda(), epilogue="float", out=out)
    want = a.cuda().float() @ codes.cuda().float().t()  # below 2^24: exact in float32
    assert (want.abs() < 2 ** 24).all() and torch.equal(out, want)


@pytest.mark.parametrize("change", [lambda lin: lin.cpu(), lambda lin: lin.double(), lambda lin: lin.half(), lambda lin: lin.bias.data.fill_(9.0)],
                         ids=["cpu", "double", "half", "in place"])
def test_layer_outlives_changes_of_the_module_it_came_from(change):
    """The module leaves the device or changes its type after quantisation, what it freed is allocated again and overwritten:
    the layer's results stay."""
    lin = torch.nn.Linear(512, 4096, device="cuda")
    layer = ops.LinearI8(lin.weight, lin.bias)
    x = torch.randn((5, 512), device="cuda").to(torch.bfloat16)
    want = layer(x)
    torch.cuda.synchronize()
    change(lin)
    over = [torch.full((4096,), float("nan"), device="cuda") for _ in range(64)]
    assert torch.equal(layer(x), want) and len(over) == 64


def test_copied_and_saved_layers():
    """A deep copy and a saved layer give the layer's bits after the original is gone and its memory overwritten."""
    import copy
    import io
    g = torch.Generator(device="cuda").manual_seed(12)
    layer = ops.LinearI8(torch.randn((700, 900), generator=g, device="cuda"), torch.randn((700,), generator=g, device="cuda"))
    x = torch.randn((40, 900), generator=g, device="cuda").to(torch.bfloat16)
    want, file = layer(x), io.BytesIO()
    torch.save(layer, file)
    again = copy.deepcopy(layer)
    layer._packed.zero_(), layer._scale.zero_(), layer._bias.zero_()
    del layer
    file.seek(0)
    for it in (again, torch.load(file, weights_only=False)):
        assert torch.equal(it(x), want)


def test_more_columns_than_a_launch_has_tiles_of_64():
    """A few rows by so many columns that the forms of 64 columns would need more threads than a launch has: a form of larger
    tiles takes them.  Every output is checked (a power of two as scale: exact)."""
    n, m = (7 << 26) + 70, 3
    codes = torch.randint(-128, 128, (n, 1), dtype=torch.int8, device="cuda")
    layer = ops.LinearI8.from_codes(codes, torch.full((n,), 0.5, device="cuda"))
    a = torch.zeros((m, 64), dtype=torch.int8, device="cuda")
    a[:, 0] = torch.tensor([1, -127, 3])
    sa, out = torch.tensor([1.0, 2.0, 0.25], device="cuda"), torch.full((m, n), float("nan"), device="cuda")
    H.check(H.lib().oasr_gemm_i8(a.data_ptr(), 64, layer.packed.data_ptr(), sa.data_ptr(), layer.scale.data_ptr(), None, None, 0,
                                 out.data_ptr(), n, m, n, 1, 1.0, H.EPI_BIAS_F32, H.current_stream_ptr()))
    for r in range(m):
        assert torch.equal(out[r], codes[:, 0].float() * float(a[r, 0]) * float(sa[r]) * 0.5)
    del layer, out, codes
    torch.cuda.empty_cache()


def test_too_many_rows_are_a_value_error():
    layer = ops.LinearI8(torch.ones((1, 1), device="cuda"))
    with pytest.raises(ValueError, match="m must be below 2.24"):
        layer(torch.zeros((1 << 24, 1), dtype=torch.bfloat16, device="cuda"))
    torch.cuda.empty_cache()
