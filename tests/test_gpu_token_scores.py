"""GPU tests of the token scores against 64-bit log-softmax, entropy and a sort by (value, index).

Bounds.  u = 2^-24.  Every exponential has an argument d rounded twice (m - z, times log2 e): relative error 2 u d + 2 u of
the instruction, and exp(-d) d <= 1 / e, so the errors of S sum to at most 4 u S (a term's weight p times 2 d u, with
p d <= log2-sized entropy: at most 2 u (H + 1) more).  Partial sums: at most 2^-24 * (terms per lane + 24) relative, 600 terms
here: 2^-14.8 in the worst case and sqrt(600) u as a rule; the bound takes 2^-17 for S and T.  log S is then within 2^-17 +
u log S, z - m and the last difference within 2 u |log p|:  |d log p| <= 2^-17 + 2^-22 |log p|, |d H| <= 2^-16 (1 + H)."""

import math

import pytest
import torch

from omnilingual_asr import _hip as H
from omnilingual_asr import ops

pytestmark = pytest.mark.gpu
INF = math.inf


def reference(z, tokens, k):
    """64-bit results of rows z [rows, vocab]: (logprobs, entropy, ids, best) with the documented special rows."""
    z = z.double().cpu()
    rows, v = z.shape
    bad = torch.isnan(z).any(1) | (z == INF).any(1)
    empty = (z == -INF).all(1)
    safe = torch.where((bad | empty)[:, None], torch.zeros_like(z), z)
    logp = torch.log_softmax(safe, 1)
    ent = -torch.where(logp == -INF, torch.zeros_like(logp), logp.exp() * logp).sum(1)
    order = torch.sort(safe, dim=1, descending=True, stable=True).indices[:, :k]
    best = logp.gather(1, order)
    ids = torch.where(best == -INF, torch.full_like(order, -1), order)
    if v < k:
        ids = torch.nn.functional.pad(ids, (0, k - v), value=-1)
        best = torch.nn.functional.pad(best, (0, k - v), value=-INF)
    t = tokens.long().cpu()
    lp = logp.gather(1, t.clamp(0, v - 1))
    lp = torch.where(empty[:, None], torch.full_like(lp, -INF), lp)
    lp = torch.where((t >= v) | bad[:, None], torch.full_like(lp, math.nan), lp)
    lp = torch.where(t < 0, torch.zeros_like(lp), lp)
    ent = torch.where(empty, torch.zeros_like(ent), ent)
    ent = torch.where(bad, torch.full_like(ent, math.nan), ent)
    ids = torch.where((bad | empty)[:, None], torch.full_like(ids, -1), ids)
    best = torch.where(empty[:, None], torch.full_like(best, -INF), best)
    best = torch.where(bad[:, None], torch.full_like(best, math.nan), best)
    return lp, ent, ids, best


def close(got, want, bound):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = (got[fine] - want[fine]).abs() - bound(want[fine])
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def check(r, z, tokens, k):
    lp, ent, ids, best = reference(z, tokens, k)
    close(r.logprobs, lp, lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
    close(r.entropy, ent, lambda w: 2.0 ** -16 * (1 + w))
    close(r.best, best, lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
    assert torch.equal(r.ids.cpu().long(), ids)


SIZES = [(1, 1, 1), (3, 2, 4), (5, 31, 5), (9, 32, 4), (17, 33, 32), (130, 100, 8), (7, 255, 3), (6, 256, 32), (5, 257, 7),
         (9, 511, 1), (4, 1000, 20), (3, 1024, 32), (3, 1025, 32), (5, 1030, 5), (70, 2000, 8), (5, 2047, 20), (4, 2048, 32), (3, 2049, 7), (33, 700, 3), (2, 4095, 9), (300, 5001, 8), (1, 8192, 32),
         (2, 16391, 20), (40, 32000, 5), (1, 50257, 20), (257, 20011, 32), (1, 131072, 8), (3, 200003, 20), (64, 70000, 0), (5, 65537, 9), (128, 66000, 3), (2, 600001, 32), (4100, 2111, 32), (4200, 9000, 5), (1030, 9001, 20), (401, 31000, 8), (600, 4999, 12)]


@pytest.mark.parametrize("rows,vocab,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_token_scores(rows, vocab, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab + k)
    pitch = vocab + rows % 5
    z = torch.full((rows, pitch), float("nan"), dtype=dtype, device="cuda")
    z[:, :vocab] = torch.randn((rows, vocab), generator=g, device="cuda") * 3
    if vocab > 8:                                   # masked tokens, and the lowest value as a mask
        drop = torch.rand((rows, vocab), generator=g, device="cuda")
        z[:, :vocab] = z[:, :vocab].masked_fill(drop < 0.2, -INF).masked_fill(drop > 0.9, torch.finfo(dtype).min)
    z = z[:, :vocab]
    tokens = torch.randint(-1, vocab, (rows, 3), generator=g, device="cuda", dtype=torch.int32)
    tokens[:, 0] = z.float().argmax(1).int()
    check(ops.token_scores(z, tokens, alternatives=k), z, tokens, k)


@pytest.mark.parametrize("vocab", [1, 5, 32, 300, 1024, 1500, 2500, 9001, 40000, 140001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_special_rows(vocab, dtype):
    """Rows that allow nothing, one token, the lowest value everywhere, NaN and infinities at the first, a middle and the
    last place, equal values throughout (more ties than the kernel keeps at once), a probability of nearly one."""
    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(dtype).min
    rows = []

    def row(base, **at):
        z = torch.full((vocab,), base) if not isinstance(base, torch.Tensor) else base.clone()
        for place, value in at.items():
            z[{"first": 0, "mid": vocab // 2, "last": vocab - 1}[place]] = value
        rows.append(z)

    noise = torch.randn((vocab,), generator=g)
    row(-INF)
    row(-INF, mid=1.5)
    row(-INF, first=low, last=low)
    row(low)
    row(low, mid=0.0)
    row(noise, first=math.nan)
    row(noise, mid=math.nan)
    row(noise, last=math.nan)
    row(math.nan)
    row(noise, last=INF)
    row(noise, first=INF, mid=-INF)
    row(INF)
    row(0.25)
    row(0.0, mid=-0.0)
    row(-3.0, last=60.0)
    row(noise, last=20.0)
    row(-1e30, first=0.0, mid=1.0)
    row(torch.linspace(-4, 4, vocab))
    row(torch.linspace(4, -4, vocab))
    row((noise * 2).round())
    z = torch.stack(rows).to(dtype).cuda()
    n = z.shape[0]
    tokens = torch.tensor([[0, vocab // 2, vocab - 1, -1, vocab, -7, 2 ** 31 - 1]] * n, dtype=torch.int32).cuda()
    for k in (0, 1, 5, 32):
        check(ops.token_scores(z, tokens, alternatives=k), z, tokens, k)
    for i in (0, 5, 12, 15):                        # alone: the form that cuts a row, where it is long
        check(ops.token_scores(z[i: i + 1], tokens[i: i + 1], alternatives=5), z[i: i + 1], tokens[i: i + 1], 5)


def test_all_equal_long_rows_take_the_lowest_indices():
    for v, rows in ((150000, 1), (150000, 300), (1024, 5)):
        r = ops.token_scores(torch.full((rows, v), -2.0, device="cuda"), alternatives=32)
        assert torch.equal(r.ids.cpu(), torch.arange(32, dtype=torch.int32).expand(rows, 32))
        assert (r.best.cpu() + math.log(v)).abs().max() < 2 ** -16 and (r.entropy.cpu() - math.log(v)).abs().max() < 2 ** -12


def test_shapes_of_inputs_and_empty_batches():
    g = torch.Generator().manual_seed(1)
    z = torch.randn((2, 3, 77), generator=g).cuda()
    tok = torch.randint(0, 77, (2, 3), generator=g, dtype=torch.int32).cuda()
    r = ops.token_scores(z, tok, alternatives=2)
    assert r.logprobs.shape == (2, 3) and r.entropy.shape == (2, 3) and r.ids.shape == (2, 3, 2) and r.best.shape == (2, 3, 2)
    check(ops.TokenScores(r.logprobs.view(6, 1), r.entropy.view(6), r.ids.view(6, 2), r.best.view(6, 2)), z.view(6, 77), tok.view(6, 1), 2)
    one = ops.token_scores(z[1, 2], tok[1, 2], alternatives=2)
    assert one.logprobs.shape == () and torch.equal(one.ids, r.ids[1, 2]) and torch.equal(one.logprobs, r.logprobs[1, 2])
    none = ops.token_scores(z)
    assert none.logprobs.shape == (2, 3, 0) and none.ids.shape == (2, 3, 0) and torch.equal(none.entropy, r.entropy)
    for empty in (ops.token_scores(z[:0], tok[:0], alternatives=2), ops.token_scores(z[:, :0], tok[:, :0], alternatives=2)):
        assert empty.logprobs.numel() == 0 and empty.ids.shape[-1] == 2
    assert ops.token_scores(z, tok[..., None].expand(2, 3, 4)).logprobs.shape == (2, 3, 4)
    for bad, text in ((lambda: ops.token_scores(z, tok[:1]), "tokens"), (lambda: ops.token_scores(z, tok.long()), "int32"),
                      (lambda: ops.token_scores(z, tok, alternatives=33), "alternatives"), (lambda: ops.token_scores(z[..., :0]), "column"),
                      (lambda: ops.token_scores(z.transpose(1, 2)[0]), "contiguous rows"), (lambda: ops.token_scores(z, tok.cpu()), "on cuda")):
        with pytest.raises(ValueError, match=text):
            bad()


def test_rows_do_not_depend_on_the_batch_and_offsets_past_32_bits():
    """The same row alone (cut over work-groups), among a few and among many agrees within the bounds; a row whose offset
    needs more than 32 bits is the row it should be."""
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn((600, 30001), generator=g, device="cuda")
    tok = torch.randint(0, 30001, (600, 2), generator=g, device="cuda", dtype=torch.int32)
    full = ops.token_scores(z, tok, alternatives=6)
    for lo, n in ((0, 1), (17, 5), (300, 200)):
        part = ops.token_scores(z[lo: lo + n], tok[lo: lo + n], alternatives=6)
        assert torch.equal(part.ids, full.ids[lo: lo + n])
        assert (part.logprobs - full.logprobs[lo: lo + n]).abs().max() <= 2 ** -16 + 2 ** -21 * 30
        assert (part.entropy - full.entropy[lo: lo + n]).abs().max() <= 2 ** -15 * 12
    far = torch.empty((1 << 32) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    rows = far.as_strided((3, 5000), (1 << 31, 1))
    rows.copy_(z[:3, :5000])
    check(ops.token_scores(rows, tok[:3] % 5000, alternatives=4), rows.float(), tok[:3] % 5000, 4)


@pytest.mark.parametrize("batch,t,vocab,pitch,width", [(1, 32, 32, 256, 32), (3, 96, 29, 256, 96), (5, 64, 200, 256, 17), (2, 50, 1500, 1501, 50)])
def test_ctc_token_scores(batch, t, vocab, pitch, width):
    g = torch.Generator().manual_seed(batch * t)
    z = torch.randn((batch, t, pitch), generator=g) * 3
    z[..., vocab:] = math.nan                       # behind the vocabulary: never read
    frames = torch.full((batch, width), -1, dtype=torch.int32)
    tokens = torch.full((batch, width), -1, dtype=torch.int32)
    for b in range(batch):
        n = (b * 13) % (width + 1)                  # counts from none to all
        frames[b, :n] = torch.randint(0, t, (n,), generator=g, dtype=torch.int32)
        tokens[b, :n] = torch.randint(0, vocab, (n,), generator=g, dtype=torch.int32)
    frames[-1, 0], tokens[-1, 0] = t, 0             # a frame that does not exist
    zd = z.cuda()
    r = ops.ctc_token_scores(zd, tokens.cuda(), frames.cuda(), vocab=vocab, alternatives=3)
    row = z[torch.arange(batch)[:, None], frames.long().clamp(0, t - 1)].reshape(batch * width, pitch)[:, :vocab]
    lp, ent, ids, best = reference(row, tokens.view(-1, 1), 3)
    absent, wrong = tokens.view(-1) < 0, frames.view(-1) >= t
    fill = lambda x, a, w: torch.where(absent.view(-1, *[1] * (x.dim() - 1)), torch.full_like(x, a),  # noqa: E731
                                       torch.where(wrong.view(-1, *[1] * (x.dim() - 1)), torch.full_like(x, w), x))
    close(r.logprobs.view(-1, 1), fill(lp, 0.0, math.nan), lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
    close(r.entropy.view(-1), fill(ent, 0.0, math.nan), lambda w: 2.0 ** -16 * (1 + w))
    close(r.best.view(-1, 3), fill(best, -INF, math.nan), lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
    assert torch.equal(r.ids.view(-1, 3).cpu().long(), fill(ids, -1, -1))


def test_scores_of_a_greedy_decode():
    """The decode's own tokens: each is the first alternative of its frame, with the same log probability."""
    g = torch.Generator().manual_seed(7)
    batch, t, vocab, pitch = 4, 160, 32, 256
    z = (torch.randn((batch, t, pitch), generator=g) * 4).cuda()
    lengths = torch.tensor([160, 1, 0, 77], dtype=torch.int32).cuda()
    tok, frm = (torch.zeros((batch, t), dtype=torch.int32, device="cuda") for _ in range(2))
    cnt = torch.zeros((batch,), dtype=torch.int32, device="cuda")
    ws = torch.zeros((batch * t,), dtype=torch.int32, device="cuda")
    H.check(H.lib().oasr_ctc_greedy(z.data_ptr(), pitch, vocab, lengths.data_ptr(), batch, t, 0, tok.data_ptr(), frm.data_ptr(),
                                    cnt.data_ptr(), ws.data_ptr(), H.current_stream_ptr()))
    r = ops.ctc_token_scores(z, tok, frm, vocab=vocab, alternatives=2)
    there = tok >= 0
    assert int(there.sum()) == int(cnt.sum()) > 100
    assert torch.equal(r.ids[..., 0], tok) and torch.equal(r.best[..., 0][there], r.logprobs[there])
    assert (r.logprobs[~there] == 0).all() and (r.entropy[~there] == 0).all() and (r.best[~there] == -INF).all()
    assert (r.best[..., 1][there] <= r.best[..., 0][there]).all() and (r.entropy[there] > 0).all()


def test_streams_and_repeated_graph_replays():
    g = torch.Generator().manual_seed(9)
    for rows, vocab in ((1, 131072), (5, 40000), (700, 3000), (33, 100)):
        a, b = (torch.randn((rows, vocab), generator=g).cuda() for _ in range(2))
        tok = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32).cuda()
        want = {0: ops.token_scores(a, tok, alternatives=4), 1: ops.token_scores(b, tok, alternatives=4)}
        torch.cuda.synchronize()
        buf, graphs, side = a.clone(), [], torch.cuda.Stream()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = ops.token_scores(buf, tok, alternatives=4)
            graphs.append((graph, out))
        for rep in range(4):
            buf.copy_((a, b)[rep & 1])
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                eager = ops.token_scores(b, tok, alternatives=4)
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(x, y) for x, y in zip(out, want[rep & 1]))
            assert all(torch.equal(x, y) for x, y in zip(eager, want[1]))


@pytest.mark.parametrize("rows,vocab", [(3, 50257), (3, 33001), (800, 20011), (2, 131075), (5, 2049), (4100, 2111), (1030, 9001), (401, 20000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_likeliest_wherever_they_lie(rows, vocab, dtype):
    """The likeliest values next to each other, at strides that meet in one thread's share (in one step and in several), in the
    last chunks and behind them: every one is found, once."""
    strides = [1, 4, 8, 1024, 2048, 4096, 8192, 16384, 7, vocab // 32]
    g = torch.Generator().manual_seed(vocab)
    for stride in strides:
        z = torch.rand((rows, vocab), generator=g) * 2
        places = []
        for r in range(rows):
            start = int(torch.randint(0, vocab, (1,), generator=g)) if r else vocab - 1 - 31 * (stride if 31 * stride < vocab else 1)
            at = torch.unique((start + stride * torch.arange(32)) % vocab)
            at = at[torch.randperm(at.numel(), generator=g)]
            z[r, at] = 8.0 + torch.arange(at.numel(), 0, -1) * 0.25       # exact in bfloat16, all different
            places.append(at)
        s = ops.token_scores(z.to(dtype).cuda(), alternatives=32)
        ids = s.ids.cpu()
        for r in range(rows):
            assert ids[r, :places[r].numel()].tolist() == places[r].tolist(), (stride, r)
            assert ids[r].unique().numel() == 32


@pytest.mark.parametrize("vocab", [2049, 2500, 9001])
def test_special_rows_among_many(vocab):
    """The special rows within thousands of others: each row's results depend on that row alone."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = torch.randn((4111, vocab), generator=g, device="cuda") * 3
    z[5] = -INF
    z[6] = -INF
    z[6, vocab - 1] = 2.0
    z[7] = torch.finfo(torch.float32).min
    z[8, 0], z[9, vocab // 2], z[10, vocab - 1] = math.nan, INF, -INF
    z[11] = 1.5
    z[12, ::2] = -INF
    z[13, vocab - 1] = 90.0
    tokens = torch.randint(0, vocab, (4111, 1), generator=g, device="cuda", dtype=torch.int32)
    at = torch.cat([torch.arange(0, 20), torch.tensor([4096, 4110])])
    many = ops.token_scores(z, tokens, alternatives=32)
    check(ops.TokenScores(*(v[at.cuda()] for v in many)), z[at.cuda()], tokens[at.cuda()], 32)


@pytest.mark.parametrize("rows,vocab", [(6, 1 << 26), (140, 1 << 20), (140, 300007), (4200, 10001), (1100, 10001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_sums_of_long_rows_do_not_drift(rows, vocab, dtype):
    """Rows of one value (z < 0) with a 0 at every 509th place (each wave then sums terms exp(z), which all round the same way):
    S = n + (V - n) exp(z), T = (V - n) exp(z) (-z).  In units of u = 2^-24, for |z| <= 5: a term is within 12, a step's sixteen
    terms add 15, the compensated sum 3, the joins over lanes, waves and parts at most 48: S and T within 78 u of themselves, 2^-17.7;
    the logarithm and the last difference add 2^-22 |log p|.  A plain sum of the 4096 terms of a lane is off by up to 2^-14.6."""
    values = [math.log(0.7), math.log(0.3), math.log(0.999), -5.0, -2.2, -0.1]
    z = torch.empty((rows, vocab), dtype=dtype, device="cuda")
    for r in range(rows):
        z[r] = values[r % 6]
    z[:, 3::509] = 0
    n = len(range(3, vocab, 509))
    at = torch.tensor([[3, 0]] * rows, dtype=torch.int32, device="cuda")
    got = ops.token_scores(z, at, alternatives=1)
    low = z[:, 0].double().cpu()
    t = (vocab - n) * torch.exp(low) * -low
    total = n + (vocab - n) * torch.exp(low)
    want = -torch.log(total)
    close(got.logprobs, torch.stack([want, low + want], 1), lambda w: 2.0 ** -17 + 2.0 ** -22 * w.abs())
    entropy = torch.log(total) + t / total
    assert ((got.entropy.double().cpu() - entropy).abs() <= 2.0 ** -17 * (1 + t / total) + 2.0 ** -22 * entropy).all()
    assert (got.ids == 3).all()


def test_sizes_past_the_limits_are_refused_as_value_errors():
    with pytest.raises(ValueError, match="2.24 rows"):
        ops.token_scores(torch.zeros((1 << 24, 1), device="cuda"))
    with pytest.raises(ValueError, match="2.30 columns"):
        ops.token_scores(torch.empty((1, (1 << 32) + 5), dtype=torch.bfloat16, device="cuda"), alternatives=2)
    torch.cuda.empty_cache()
