"""Refusals of the 8-bit integer operators, made before anything is launched (no GPU needed), and the host-side quantiser."""

import numpy
import pytest
import torch

from omnilingual_asr import _hip, ops
from omnilingual_asr.weights import quantize_rows_i8
from tests.i8_tools import quantize64

A = 1 << 20        # a plausible, aligned address: every call below is refused before it would be used


def _gemm(**kw):
    d = dict(a=A, lda=64, w=A, sa=A, sw=A, bias=None, resid=None, ldr=64, c=A, ldc=64, m=4, n=64, k=64, alpha=1.0, epi=0)
    d.update(kw)
    return _hip.lib().oasr_gemm_i8(d["a"], d["lda"], d["w"], d["sa"], d["sw"], d["bias"], d["resid"], d["ldr"], d["c"], d["ldc"],
                                   d["m"], d["n"], d["k"], d["alpha"], d["epi"], None)


def _linear(**kw):
    d = dict(x=A, ldx=64, w=A, sw=A, bias=None, resid=None, ldr=64, c=A, ldc=64, m=4, n=64, k=64, alpha=1.0, epi=0, ws=A, bytes=1 << 20)
    d.update(kw)
    return _hip.lib().oasr_linear_i8(d["x"], d["ldx"], d["w"], d["sw"], d["bias"], d["resid"], d["ldr"], d["c"], d["ldc"], d["m"],
                                     d["n"], d["k"], d["alpha"], d["epi"], d["ws"], d["bytes"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(n=0), "positive"), (dict(k=0), "positive"), (dict(m=-1), "positive"), (dict(k=131073, lda=131136), "131072"),
    (dict(epi=5), "epilogue"), (dict(epi=-1), "epilogue"), (dict(epi=2, n=48), "multiple of 32"), (dict(ldc=63), "ldc"),
    (dict(epi=3, resid=A, ldr=63), "ldr"), (dict(w=None), "null"), (dict(sw=None), "null"), (dict(c=None), "null"), (dict(epi=3), "resid"), (dict(w=A + 8), "aligned"),
    (dict(c=A + 1), "aligned"), (dict(epi=4, c=A + 2), "aligned"), (dict(m=1 << 31), "2^31"),
])
def test_product_refusals(kw, text):
    for call, name in ((_gemm, "gemm_i8"), (_linear, "linear_i8")):
        assert call(**kw) == -1
        msg = _hip.lib().oasr_last_error().decode()
        assert name in msg and text in msg, msg


def test_operand_refusals():
    L = _hip.lib()
    assert _gemm(lda=48) == -1 and b"lda" in L.oasr_last_error()
    assert _gemm(lda=72) == -1 and _gemm(k=65) == -1 and _gemm(a=None) == -1 and _gemm(a=A + 8) == -1 and _gemm(sa=None) == -1
    assert _linear(ldx=63) == -1 and b"ldx" in L.oasr_last_error()
    many = dict(m=300, k=2000, ldx=2000)
    assert _linear(x=None) == -1 and _linear(ws=None, **many) == -1 and _linear(ws=A + 16, **many) == -1 and _linear(x=A + 1) == -1
    need = L.oasr_linear_i8_workspace_bytes(300, 64, 2000)
    assert need == 300 * 2048 + 1280 and _linear(bytes=need - 1, **many) == -2 and b"workspace" in L.oasr_last_error()
    assert L.oasr_linear_i8_workspace_bytes(1, 64, 4096) == 0 and L.oasr_linear_i8_workspace_bytes(0, 64, 64) == 0
    assert _gemm(m=0, a=None, w=None, c=None) == 0 and _linear(m=0, x=None, ws=None) == 0     # nothing to do
    q = lambda x=A, ldx=64, rows=4, k=64, y=A, ldy=64, s=A: L.oasr_quant_i8_rows(x, ldx, rows, k, y, ldy, s, None)
    assert q(ldx=63) == -1 and q(ldy=56) == -1 and q(k=65, ldx=65) == -1 and q(k=0) == -1 and q(rows=-1) == -1
    assert q(x=None) == -1 and q(y=A + 8) == -1 and q(s=A + 2) == -1 and q(rows=0, x=None) == 0
    ln = lambda x=A, d=512, rows=4, y=A: L.oasr_layernorm_i8(x, A, A, y, A, rows, d, 1e-5, 0, None)
    assert ln(d=160) == -1 and b"unsupported width" in L.oasr_last_error()
    assert ln(x=None) == -1 and ln(x=A + 4) == -1 and ln(y=A + 4) == -1 and ln(rows=-1) == -1 and ln(rows=0) == 0
    assert L.oasr_layernorm2_i8(A, A, A, None, A, A, A, 4, 512, 1e-5, None) == -1
    pack = lambda w=A, ldw=64, n=16, k=64, out=2 * A: L.oasr_gemm_pack_w_i8(w, ldw, n, k, out, None)
    assert pack(w=None) == -1 and pack(out=A) == -1 and pack(ldw=63) == -1 and pack(n=0) == -1 and pack(out=2 * A + 8) == -1
    assert pack(k=131073, ldw=131073) == -1


def test_sizes_beyond_a_launch_are_refused():
    """A launch has fewer than 2^32 threads: what would need more is refused, not cut short."""
    L = _hip.lib()
    text = lambda: L.oasr_last_error().decode()
    assert L.oasr_quant_i8_rows(A, 16, 1 << 24, 16, A, 64, A, None) == -1 and "2^24" in text()
    assert L.oasr_layernorm_i8(A, A, A, A, A, (1 << 26) - 4, 256, 1e-5, 0, None) == -1 and "2^26" in text()
    assert L.oasr_gemm_pack_w_i8(A, 64, (1 << 30) + 1, 64, 2 * A, None) == -1 and "64 GiB" in text()
    assert _gemm(m=(1 << 31) - 1, n=(1 << 31) - 1, ldc=1 << 31) == -1 and "too large" in text()
    assert _linear(m=1, n=1 << 28, ldc=1 << 28) == -1 and "too large" in text()
    assert _linear(m=1 << 24, ldx=2048, k=2048, bytes=1 << 50) == -1 and "2^24" in text()


def test_packed_bytes():
    f = _hip.lib().oasr_gemm_i8_packed_bytes
    assert f(1, 1) == 1024 and f(16, 64) == 1024 and f(17, 64) == 2048 and f(16, 65) == 2048 and f(0, 4) == 0 and f(4, -1) == 0


def test_tensor_refusals_without_a_device():
    w, x = torch.zeros((32, 64)), torch.zeros((3, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="HIP device"):
        ops.LinearI8(w)
    with pytest.raises(ValueError, match="float tensor"):
        ops.LinearI8(w.to(torch.int8))
    with pytest.raises(ValueError, match=r"\[out, in\]"):
        ops.LinearI8.from_codes(torch.zeros((4,), dtype=torch.int8), torch.ones((4,)))
    with pytest.raises(ValueError, match="int8"):
        ops.LinearI8.from_codes(w, torch.ones((32,)))
    with pytest.raises(ValueError, match="one column"):
        ops.LinearI8(torch.zeros((32, 0)))
    with pytest.raises(ValueError, match=r"\[out, in\]"):
        ops.LinearI8.from_codes(None, None)
    layer = ops.LinearI8.__new__(ops.LinearI8)
    layer.device, layer.in_features, layer.out_features = torch.device("cpu"), 64, 32
    with pytest.raises(ValueError, match="HIP device"):
        layer(x)
    with pytest.raises(ValueError, match="bfloat16"):
        layer(x.float())


def test_host_quantiser_is_the_definition():
    g = torch.Generator().manual_seed(3)
    w = torch.randn((37, 129), generator=g)
    w[5] = 0
    codes, scale = quantize_rows_i8(w)
    want, s = quantize64(w)
    assert codes.dtype == torch.int8 and torch.equal(codes.double(), want) and torch.equal(scale, s.float())
    assert scale[5] == 1.0 and int(codes.abs().max()) == 127
    w[1, 3], w[2, 0] = float("nan"), float("inf")
    codes, scale = quantize_rows_i8(w)
    assert torch.isnan(scale[1]) and torch.isinf(scale[2]) and (codes[1:3] == 0).all() and torch.isfinite(scale[3:]).all()


def test_pipeline_takes_one_kind_of_8_bit_weights():
    from omnilingual_asr import Pipeline
    with pytest.raises(ValueError, match="exclude"):
        Pipeline(fp8=True, int8=True)
    assert Pipeline(int8=True).gemini._int8


def test_encoder_takes_one_kind_of_8_bit_weights():
    """Handles are host memory: the refusals need no device."""
    import ctypes as C
    L = _hip.lib()
    cfg = _hip.EncoderConfig(160, 512, 1024, 8, 1, 31, 64, 8, 1e-5)
    handle = C.c_void_p()
    assert L.oasr_encoder_create(C.byref(cfg), C.byref(_hip.TopWeights()), (_hip.LayerWeights * 1)(), C.byref(handle)) == 0
    try:
        full = {k: A for k in _hip.FP8_FIELDS}
        before = L.oasr_encoder_workspace_bytes(handle, 1, 32)
        assert L.oasr_encoder_set_int8(None, None) == -1
        assert L.oasr_encoder_set_int8(handle, (_hip.LayerInt8Weights * 1)()) == -1 and b"layer 0" in L.oasr_last_error()
        assert L.oasr_encoder_set_int8(handle, (_hip.LayerInt8Weights * 1)(_hip.LayerInt8Weights(**full))) == 0
        assert L.oasr_encoder_workspace_bytes(handle, 1, 32) > before
        assert L.oasr_encoder_set_fp8(handle, (_hip.LayerFp8Weights * 1)(_hip.LayerFp8Weights(**full))) == -1
        assert b"int8" in L.oasr_last_error()
        assert L.oasr_encoder_set_int8(handle, None) == 0 and L.oasr_encoder_workspace_bytes(handle, 1, 32) == before
        assert L.oasr_encoder_set_fp8(handle, (_hip.LayerFp8Weights * 1)(_hip.LayerFp8Weights(**full))) == 0
        assert L.oasr_encoder_set_int8(handle, (_hip.LayerInt8Weights * 1)(_hip.LayerInt8Weights(**full))) == -1
    finally:
        L.oasr_encoder_destroy(handle)


@pytest.fixture
def recorded(monkeypatch):
    """Layers on host tensors: what a call would hand to the library, as (name, arguments), instead of the call."""
    calls = []
    monkeypatch.setattr(ops, "_rows", lambda t, what, dtypes: (t, t.numel() // t.shape[-1], t.shape[-1], t.shape[-1]))
    monkeypatch.setattr(ops, "_call", lambda name, device, *args: calls.append((name, args)))
    return calls


def _handed_over(layer, calls):
    """The addresses of weights, scale and bias that a call on `layer` passes."""
    del calls[:]
    layer(torch.zeros((1, layer.in_features), dtype=torch.bfloat16))
    (name, args), = calls
    assert name == "oasr_linear_i8"
    return args[2:5]


def test_layer_reads_its_own_memory_when_a_module_moves(recorded):
    """Module.to() and the like put new storage under the same Parameter object and free the old one: a layer made from a
    module's Parameters reads memory of its own, whatever happens to them."""
    lin = torch.nn.Linear(64, 32)
    layer = ops.LinearI8(lin.weight, lin.bias)
    scale = torch.rand(32)
    other = ops.LinearI8.from_codes(torch.ones((32, 64), dtype=torch.int8), scale, lin.bias)
    kept = lin.bias.detach().clone()
    before = _handed_over(layer, recorded)
    foreign = {lin.bias.data_ptr(), scale.data_ptr()}
    lin.double()
    for it in (layer, other):
        own = _handed_over(it, recorded)
        assert own == (it.packed.data_ptr(), it.scale.data_ptr(), it.bias.data_ptr())
        assert not foreign & set(own) and lin.bias.data_ptr() not in own
        assert torch.equal(it.bias, kept) and it.bias.dtype == torch.float32 and not it.bias.requires_grad
    assert _handed_over(layer, recorded) == before and torch.equal(other.scale, scale)


@pytest.mark.parametrize("name", ["scale", "bias", "packed"])
def test_buffers_of_a_layer_cannot_be_assigned(recorded, name):
    """An assigned tensor would not be what the kernels read."""
    layer = ops.LinearI8(torch.ones((32, 64)), torch.ones(32))
    before = _handed_over(layer, recorded)
    with pytest.raises(AttributeError):
        setattr(layer, name, torch.zeros(32))
    getattr(layer, name).data = torch.zeros(32)          # of the alias: the layer keeps its own
    assert _handed_over(layer, recorded) == before == (layer.packed.data_ptr(), layer.scale.data_ptr(), layer.bias.data_ptr())


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle"])
def test_copies_of_a_layer_read_their_own_memory(recorded, how):
    """A copy passes the addresses of its own buffers, not those of the layer that it was made from."""
    import copy
    import pickle
    again = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda t: pickle.loads(pickle.dumps(t))}[how]
    for bias in (torch.rand(32), None):
        layer = ops.LinearI8(torch.rand((32, 64)), bias)
        layer._packed.copy_(torch.arange(2048) % 127)
        it = again(layer)
        got, mine = _handed_over(it, recorded), _handed_over(layer, recorded)
        assert got == (it.packed.data_ptr(), it.scale.data_ptr(), None if bias is None else it.bias.data_ptr())
        assert (got == mine) == (how == "copy")
        assert torch.equal(it.packed, layer.packed) and torch.equal(it.scale, layer.scale)
        assert (it.device, it.out_features, it.in_features) == (layer.device, 32, 64)


def test_a_loaded_layer_has_to_be_on_a_device_and_whole(monkeypatch, recorded):
    import pickle
    layer = ops.LinearI8(torch.rand((32, 64)), torch.rand(32))
    state = layer.__getstate__()
    for change in (dict(shape=(32, 65)), dict(shape=(33, 64)), dict(scale=state["scale"][:31]), dict(bias=state["bias"].double())):
        with pytest.raises(ValueError):
            ops.LinearI8.__new__(ops.LinearI8).__setstate__({**state, **change})
    saved = pickle.dumps(layer)
    monkeypatch.undo()                                   # host tensors again, as loading onto the host makes them
    with pytest.raises(ValueError, match="HIP device"):
        pickle.loads(saved)


def test_arguments_of_other_types_are_value_errors(recorded):
    """Before anything is launched, in the normalising call too."""
    layer = ops.LinearI8(torch.rand((32, 256)), torch.rand(32))
    x, v = torch.zeros((2, 256), dtype=torch.bfloat16), torch.ones(256)
    del recorded[:]
    for bad in ("0.5", None, [1.0], 1j, torch.tensor(0.5)):
        for call in (lambda: layer(x, alpha=bad), lambda: layer.normed(x.float(), v, v, alpha=bad),
                     lambda: layer.normed(x.float(), v, v, eps=bad)):
            with pytest.raises(ValueError, match="must be a number"):
                call()
    for bad in (["bias"], None, 0, {}):
        with pytest.raises(ValueError, match="epilogue must be"):
            layer(x, epilogue=bad)
    assert not recorded
    for good in (1, 0.5, numpy.float32(2)):
        layer(x, alpha=good)
    assert len(recorded) == 3


def test_sizes_that_the_library_refuses_are_value_errors(monkeypatch):
    """What only the C call knows to be too large arrives as the refusal it is; a failing launch stays an OasrError."""
    lib = _hip.lib()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_hip, "stream_ptr", lambda index: None)
    monkeypatch.setattr(lib, "oasr_linear_i8", lambda stream: lib.oasr_quant_i8_rows(A, 16, 1 << 24, 16, A, 64, A, stream))
    with pytest.raises(ValueError, match="rows must be below"):
        ops._call("oasr_linear_i8", torch.device("cuda", 0))
    monkeypatch.setattr(lib, "oasr_linear_i8", lambda stream: -3)
    with pytest.raises(_hip.OasrError):
        ops._call("oasr_linear_i8", torch.device("cuda", 0))


def test_packed_weights_survive_a_module_that_moves():
    """Weights that are Parameters of the wanted type are packed without a copy: their memory has to stay when the module they
    belong to changes its type, since the encoder keeps addresses."""
    from omnilingual_asr.weights import GEOMETRIES, init_random_weights, pack_for_device
    g = GEOMETRIES["GTINY"]
    w = init_random_weights(g, 1)
    held = torch.nn.ParameterDict({"fp_b": w["fp_b"], "bo": w["layers"][0]["bo"]})
    w["fp_b"], w["layers"][0]["bo"] = held["fp_b"], held["bo"]
    packed = pack_for_device(w, g, "cpu", int8=True)
    tensors = [packed["top"]["fp_b"], packed["layers"][0]["bo"]]
    before = [(t.data_ptr(), t.clone()) for t in tensors]
    held.double()
    for t, (address, values) in zip(tensors, before):
        assert t.data_ptr() == address and t.dtype == torch.float32 and torch.equal(t, values) and not t.requires_grad
