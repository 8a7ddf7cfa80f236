"""Refusals of the token scores, made before anything is launched (no GPU needed)."""

import numpy
import pytest
import torch

from omnilingual_asr import _hip, ops

A = 1 << 20


def _scores(**kw):
    d = dict(z=A, dtype=0, ld=64, rows=4, vocab=60, tok=A, given=1, lp=A, ent=A, top=2, ids=A, best=A, ws=None, bytes=0)
    d.update(kw)
    return _hip.lib().oasr_token_scores(d["z"], d["dtype"], d["ld"], d["rows"], d["vocab"], d["tok"], d["given"], d["lp"], d["ent"],
                                        d["top"], d["ids"], d["best"], d["ws"], d["bytes"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 25), "rows"), (dict(rows=1 << 24), "rows"), (dict(vocab=0), "vocab"),
    (dict(vocab=1 << 30, ld=1 << 30), "vocab"), (dict(ld=59), "ld"), (dict(given=-1), "given"), (dict(top=-1), "top"),
    (dict(top=33), "top"), (dict(z=None), "null"), (dict(tok=None), "null"), (dict(lp=None), "null"), (dict(ids=None), "null"),
    (dict(best=None), "null"), (dict(z=A + 2), "misaligned"), (dict(dtype=1, z=A + 1), "misaligned"), (dict(ent=A + 2), "misaligned"),
])
def test_refusals(kw, text):
    assert _scores(**kw) == -1
    msg = _hip.lib().oasr_last_error().decode()
    assert "token_scores" in msg and text in msg, msg


def test_workspace_protocol():
    L = _hip.lib()
    size = L.oasr_token_scores_workspace_bytes
    assert size(0, 50000, 4) == 0 and size(4, 1000, 4) == 0 and size(4096, 50000, 4) == 0
    need = size(1, 131072, 8)
    assert need > 0
    big = dict(rows=1, vocab=131072, ld=131072, top=8)
    assert _scores(**big, ws=A, bytes=need - 1) == -2 and b"workspace needs" in L.oasr_last_error()
    assert _scores(**big, ws=A + 64, bytes=need) == -1 and _scores(**big, ws=None, bytes=need) == -1
    assert _scores(rows=0, z=None) == 0


def test_ctc_refusals():
    def call(**kw):
        d = dict(z=A, ld=64, vocab=60, batch=2, t_pad=32, tok=A, frm=A, width=32, lp=A, top=2, ids=A)
        d.update(kw)
        return _hip.lib().oasr_ctc_token_scores(d["z"], 0, d["ld"], d["vocab"], d["batch"], d["t_pad"], d["tok"], d["frm"], d["width"],
                                                d["lp"], A, d["top"], d["ids"], A, None, 0, None)
    for kw in (dict(frm=None), dict(tok=None), dict(lp=None), dict(batch=-1), dict(t_pad=0), dict(width=-1), dict(vocab=65),
               dict(top=40), dict(ids=None), dict(width=1 << 31), dict(width=1 << 24), dict(frm=A + 1)):
        assert call(**kw) == -1, kw
        assert b"ctc_token_scores" in _hip.lib().oasr_last_error()
    assert call(batch=0, z=None) == 0 and call(width=0, z=None) == 0


def test_tensor_refusals_without_a_device():
    z = torch.zeros((3, 40))
    with pytest.raises(ValueError, match="HIP device"):
        ops.token_scores(z)
    with pytest.raises(ValueError, match="must be a"):
        ops.token_scores(z.half())
    with pytest.raises(ValueError, match="contiguous tensor"):
        ops.ctc_token_scores(z, torch.zeros((3, 4), dtype=torch.int32), torch.zeros((3, 4), dtype=torch.int32))


def test_sizes_past_the_calls_32_bits_are_refused(monkeypatch):
    """A vocabulary or a batch past 2^32 must not reach the library as its low 32 bits (shapes alone: no memory behind them)."""
    monkeypatch.setattr(ops, "_rows", lambda t, what, dtypes: (t, t.numel() // t.shape[-1], t.shape[-1], t.shape[-1]))
    reached = []
    monkeypatch.setattr(ops, "_call", lambda name, device, *args: reached.append((name, args)))
    meta = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    i32 = lambda *shape: meta(*shape, dtype=torch.int32)  # noqa: E731
    for call in (lambda: ops.token_scores(meta(1, (1 << 32) + 5)), lambda: ops.token_scores(meta(2, 1 << 30)),
                 lambda: ops.token_scores(meta(1 << 24, 3)), lambda: ops.token_scores(meta(1, 5), i32(1, (1 << 32) + 1)),
                 lambda: ops.ctc_token_scores(meta((1 << 32) + 1, 1, 1), i32((1 << 32) + 1, 1), i32((1 << 32) + 1, 1)),
                 lambda: ops.ctc_token_scores(meta(1, 2, (1 << 32) + 5), i32(1, 2), i32(1, 2)),
                 lambda: ops.ctc_token_scores(meta(2, 4, 5), i32(2, 1 << 23), i32(2, 1 << 23))):
        with pytest.raises(ValueError, match="fewer than"):
            call()
    assert not reached
    ops.token_scores(meta(3, (1 << 30) - 1), i32(3, 7))
    ops.ctc_token_scores(meta(2, 4, (1 << 32) + 5), i32(2, 3), i32(2, 3), vocab=100)      # a pitch is 64 bits wide
    assert [name for name, _ in reached] == ["oasr_token_scores", "oasr_ctc_token_scores"]


def test_counts_of_other_types_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_rows", lambda t, what, dtypes: (t, t.numel() // t.shape[-1], t.shape[-1], t.shape[-1]))
    reached = []
    monkeypatch.setattr(ops, "_call", lambda name, device, *args: reached.append(args))
    z, t = torch.zeros((1, 4, 9)), torch.zeros((1, 4), dtype=torch.int32)
    for bad in (2.0, "2", None, [2], torch.tensor(2)):
        for call in (lambda: ops.token_scores(z, alternatives=bad), lambda: ops.ctc_token_scores(z, t, t, alternatives=bad)):
            with pytest.raises(ValueError, match="integer"):
                call()
    for bad in (3.7, "9"):
        with pytest.raises(ValueError, match="integer"):
            ops.ctc_token_scores(z, t, t, vocab=bad)
    assert not reached
    assert ops.ctc_token_scores(z, t, t, vocab=numpy.int64(5), alternatives=numpy.int32(2)).ids.shape == (1, 4, 2) and len(reached) == 1
