"""The int8 encoder, operator by operator: each LayerNorm, quantisation and projection of a block is given the device's own input
of that operator and compared with the definition in 64 bits, within the bounds that tests/i8_tools.py derives (the sums are
exact, so nothing but single roundings is left), and the states at the end of the chain are bit for bit those of
`oasr_encoder_forward`, which therefore runs these operators on these operands and no others.

A comparison of whole blocks with an emulating oracle cannot do this: values next to a rounding step fall on either side, and
two correct implementations end about as far apart as the quantisation itself moves them.  Parity unpinned against the
reference, which has no encoder."""

import dataclasses
import math

import pytest
import torch

from omnilingual_asr import _hip as H
from omnilingual_asr.weights import ATTENTION_Q_SCALE, GEOMETRIES, init_random_weights, pack_for_device
from tests.i8_tools import assert_within, finish64, product64, quantize64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPILOGUES = {H.EPI_BIAS_BF16: "bias", H.EPI_BIAS_SWISH_BF16: "swish", H.EPI_GLU_BF16: "glu", H.EPI_RESIDUAL_F32: "residual"}


def norm64(x, w, b, eps, swish=False):
    """LayerNorm (and Swish) in 64 bits, and how far a float32 evaluation may be.  The mean is a tree of at most 24 additions:
    within 24 u mean|x|, and mean|x| <= c std with c = sqrt(1 + mean^2 / var); x - mean rounds once more; rstd is good to
    15 u; the affine map adds three roundings.  Swish: slope at most 1.1, and 2^-16 of the value for exponential and reciprocal."""
    x, w, b = x.double(), w.double(), b.double()
    mean, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    hat, c = (x - mean) / torch.sqrt(var + eps), torch.sqrt(1 + mean ** 2 / (var + eps))
    v = hat * w + b
    off = U * (w.abs() * (25 * c + 1) + 16 * (hat * w).abs() + 3 * (v.abs() + b.abs()))
    return (v * torch.sigmoid(v), 1.1 * off + 2.0 ** -16 * v.abs()) if swish else (v, off)


def check_rows(q, s, v, off):
    """Codes and scales of rows v known to within `off`: a scale within the bound / 127 and its own roundings, a code within half a
    step, what `off` is worth in steps and 2^-16 for the two roundings of the quotient."""
    top = s.double()[:, None] * 127
    assert ((top[:, 0] - v.abs().amax(1)).abs() <= off.amax(1) + 2.0 ** -22 * top[:, 0]).all()
    assert ((q.double() - 127 * v / top).abs() <= 0.5 + 127 * off / top + 2.0 ** -16).all()
    assert (q.abs().amax(1) == 127).all()


def float_weights(L, g):
    """The eight matrices of a block as the encoder multiplies them: q rows scaled, values and gates in groups of 16."""
    d, q_scale = g.d_model, ATTENTION_Q_SCALE / math.sqrt(g.head_dim)
    order = torch.cat([torch.cat([torch.arange(16) + 16 * i, d + torch.arange(16) + 16 * i]) for i in range(d // 16)])
    return {"ffn1_w1": L["ffn1_w1"], "ffn1_w2": L["ffn1_w2"], "ffn2_w1": L["ffn2_w1"], "ffn2_w2": L["ffn2_w2"], "wo": L["wo"], "pw2": L["pw2"],
            "wqkv": torch.cat([L["wq"] * q_scale, L["wk"], L["wv"]]), "pw1": L["pw1"][order]}


class Chain:
    """The operators of `oasr_encoder_forward` one by one on device buffers, each checked on the rows that hold frames."""

    def __init__(self, g, live, rows):
        self.g, self.live, self.rows, self.checked = g, live, rows, []
        self.lib, self.st = H.lib(), H.current_stream_ptr()

    def new(self, cols, dtype):
        return torch.zeros((self.rows, cols), dtype=dtype, device="cuda")

    def use(self, P, W):
        """A block's weights: as the package lays them out, and codes and scales of the float matrices from the definition."""
        self.P, self.W, self.packed = P, {}, {}
        for name, m in W.items():
            codes, scale = (t.cuda() for t in quantize64(m))
            assert torch.equal(P[name + "_q"].double(), codes) and torch.equal(P[name + "_s"], scale.float())
            self.W[name] = codes, scale.float()
            n, k = m.shape
            out = torch.empty((int(self.lib.oasr_gemm_i8_packed_bytes(n, k)),), dtype=torch.int8, device="cuda")
            H.check(self.lib.oasr_gemm_pack_w_i8(P[name + "_q"].data_ptr(), k, n, k, out.data_ptr(), self.st))
            self.packed[name] = out

    def norm(self, x, name, rows=None, swish=False):
        d, rows = self.g.d_model, rows or self.rows
        q, s, w, b = self.new(d, torch.int8), self.new(1, torch.float32)[:, 0], self.P[name + "_w"], self.P[name + "_b"]
        H.check(self.lib.oasr_layernorm_i8(x.data_ptr(), w.data_ptr(), b.data_ptr(), q.data_ptr(), s.data_ptr(), rows, d, self.g.ln_eps,
                                           int(swish), self.st))
        n = self.live
        check_rows(q[:n], s[:n], *norm64(x[:n], w, b, self.g.ln_eps, swish))
        self.checked.append(name)
        return q, s

    def quantised(self, a):
        k = a.shape[1]
        q, s = self.new(k, torch.int8), self.new(1, torch.float32)[:, 0]
        H.check(self.lib.oasr_quant_i8_rows(a.data_ptr(), k, self.rows, k, q.data_ptr(), k, s.data_ptr(), self.st))
        want, scale = quantize64(a)
        assert torch.equal(q.double(), want) and ((s.double() - scale).abs() <= 2 * U * scale).all()
        return q, s

    def project(self, operand, name, epi, bias=None, resid=None, alpha=1.0):
        q, s = operand
        codes, sw = self.W[name]
        n, k = codes.shape
        b = None if bias is None else self.P[bias]
        cols = n // 2 if epi == H.EPI_GLU_BF16 else n
        c = self.new(cols, torch.float32 if epi == H.EPI_RESIDUAL_F32 else torch.bfloat16) if resid is None else resid.clone()
        H.check(self.lib.oasr_gemm_i8(q.data_ptr(), k, self.packed[name].data_ptr(), s.data_ptr(), self.P[name + "_s"].data_ptr(),
                                      None if b is None else b.data_ptr(), None if resid is None else c.data_ptr(), n, c.data_ptr(), cols,
                                      self.rows, n, k, alpha, epi, self.st))
        m = self.live
        before = None if resid is None else resid[:m]
        p = product64(q[:m], s[:m], codes, sw)
        assert_within(c[:m], *finish64(p, b, EPILOGUES[epi], before, alpha))
        # what the bound is worth: a weight scale that is off by 2 % does not pass
        with pytest.raises(AssertionError):
            assert_within(c[:m], *finish64(1.02 * p, b, EPILOGUES[epi], before, alpha))
        self.checked.append(name)
        return c

    def block(self, x, lengths, b, t_pad, operand, after):
        """One block on the residual stream x; `operand`: the rows that the block before left for the first projection (None in the
        first block), `after`: the next block's layout (None behind the last)."""
        g, P, lib, st = self.g, self.P, self.lib, self.st
        d, eps = g.d_model, g.ln_eps
        operand = self.norm(x, "ffn1_ln") if operand is None else operand
        hid = self.project(operand, "ffn1_w1", H.EPI_BIAS_SWISH_BF16, "ffn1_b1")
        x = self.project(self.quantised(hid), "ffn1_w2", H.EPI_RESIDUAL_F32, "ffn1_b2", x, 0.5)
        qkv = self.project(self.norm(x, "attn_ln"), "wqkv", H.EPI_BIAS_BF16, "bqkv")
        ctx = self.new(d, torch.bfloat16)
        H.check(lib.oasr_attention_relkey(qkv.data_ptr(), P["dist_emb"].data_ptr(), lengths.data_ptr(), ctx.data_ptr(), b, t_pad, g.n_heads,
                                          g.head_dim, g.left_max, g.right_max, st))
        x = self.project(self.quantised(ctx), "wo", H.EPI_RESIDUAL_F32, "bo", x)
        glu = self.project(self.norm(x, "conv_ln"), "pw1", H.EPI_GLU_BF16)
        if d in (512, 1024, 2048):
            conv = self.new(d, torch.bfloat16)
            H.check(lib.oasr_dwconv_ln_swish(glu.data_ptr(), P["dw"].data_ptr(), P["dw_ln_w"].data_ptr(), P["dw_ln_b"].data_ptr(),
                                             conv.data_ptr(), b, t_pad, d, g.conv_kernel, eps, st))
            operand = self.quantised(conv)
        else:
            conv = self.new(d, torch.float32)
            H.check(lib.oasr_dwconv_causal(glu.data_ptr(), P["dw"].data_ptr(), conv.data_ptr(), b, t_pad, d, g.conv_kernel, st))
            operand = self.norm(conv, "dw_ln", rows=self.live, swish=True)
        x = self.project(operand, "pw2", H.EPI_RESIDUAL_F32, None, x)
        hid = self.project(self.norm(x, "ffn2_ln"), "ffn2_w1", H.EPI_BIAS_SWISH_BF16, "ffn2_b1")
        x = self.project(self.quantised(hid), "ffn2_w2", H.EPI_RESIDUAL_F32, "ffn2_b2", x, 0.5)
        n, w, bb = self.live, P["final_ln_w"], P["final_ln_b"]
        v, off = norm64(x[:n], w, bb, eps)
        if after is None:
            H.check(lib.oasr_layernorm(x.data_ptr(), w.data_ptr(), bb.data_ptr(), x.data_ptr(), self.rows, d, d, eps, 0, 0, st))
            operand = None
        else:
            q, s = self.new(d, torch.int8), self.new(1, torch.float32)[:, 0]
            w2, b2 = after["ffn1_ln_w"], after["ffn1_ln_b"]
            H.check(lib.oasr_layernorm2_i8(x.data_ptr(), w.data_ptr(), bb.data_ptr(), w2.data_ptr(), b2.data_ptr(), q.data_ptr(), s.data_ptr(),
                                           self.rows, d, eps, st))
            check_rows(q[:n], s[:n], *norm64(x[:n], w2, b2, eps))
            operand = q, s
        assert ((x[:n].double() - v).abs() <= off).all()
        return x, operand


@pytest.mark.parametrize("name,ffn", [("GTINY", None), ("G300", None), ("G7B", 2048)])
def test_int8_blocks_operator_by_operator(name, ffn):
    """Two blocks (so the double LayerNorm of a block boundary is among the operators) at d = 512, d = 1024 and d = 4096, where the
    convolution branch ends in LayerNorm and Swish straight to int8 rows; ragged batch of 102 + 64 frames."""
    from omnilingual_asr.engine_hip import HipEngine
    from tests.test_gpu_ops import synth_pcm
    g = GEOMETRIES[name]
    g = dataclasses.replace(g, n_layers=2, ffn_dim=ffn or g.ffn_dim)
    w = init_random_weights(g, 41)
    n_valid = [33000, 21000]
    pcm = synth_pcm(2, 33000, seed=8)
    pcm[1, 21000:] = 0
    eng = HipEngine(g, weights=w, int8=True)
    feats, lengths = eng.features(pcm.cuda(), torch.tensor(n_valid, dtype=torch.int32, device="cuda"))
    b, t_pad, _ = feats.shape
    buf = eng._get_buffers(b, 33000)
    eng.encode_features(feats, lengths, 0, buf)
    x = buf["out"].clone()                              # the residual stream behind the input projection
    want = eng.encode_features(feats, lengths, -1, buf).clone()

    layers = pack_for_device(w, g, "cuda", int8=True)["layers"]
    chain, operand = Chain(g, b * t_pad, buf["rows"]), None
    for l in range(2):
        chain.use(layers[l], float_weights(w["layers"][l], g))
        x, operand = chain.block(x, lengths, b, t_pad, operand, layers[1] if l == 0 else None)
    got = x[: b * t_pad].view(b, t_pad, -1)
    for i in range(b):
        n = int(lengths[i])
        assert n > 60 and torch.equal(got[i, :n], want[i, :n])
    assert len(chain.checked) == 2 * 8 + (2 * (3 if ffn is None else 4) + 1)
    eng.close()


def test_int8_through_all_blocks():
    """The 300M geometry through its whole depth, distance from the float32 oracle and from the one that rounds and quantises where
    the device does, after every block.  What to expect: e4m3 operands cost 3.6e-2 k^0.4 at most after k blocks (the 7B geometry,
    tests/test_gpu_depth.py), and 8-bit integers 0.0093 per product where e4m3 costs 0.037 by arithmetic, or 0.29 of e4m3 as the
    smallest geometry shows after two blocks (1.06e-2 against 3.6e-2): 0.3 x 3.6e-2 k^0.4 here, against both oracles."""
    from tools.depth_parity import depth_curves
    g = GEOMETRIES["G300"]
    curve = depth_curves(g, [33000, 21000], fp8=False, int8=True, weights=init_random_weights(g, 43))
    for k, rel32, _, rel_emu, _ in curve:
        print("%2d blocks: float32 %.2e, emulation %.2e" % (k, rel32, rel_emu), flush=True)
    for k, rel32, _, rel_emu, _ in curve[1:]:
        assert rel32 <= 1.08e-2 * k ** 0.4 and rel_emu <= 1.08e-2 * k ** 0.4, (k, rel32, rel_emu)
        assert rel32 > 3e-3, ("int8 mode is on", k, rel32)
    assert curve[g.n_layers][1] - curve[g.n_layers // 2][1] < curve[g.n_layers // 2][1] - curve[0][1]      # no run-away
