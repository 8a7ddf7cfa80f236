"""Cases of the 8-bit integer projections and of the token scores: their inputs, the same mathematics in elementary
torch operations, and the definition in 64 bits.

A projection takes float rows x, gives every row its scale s = max|row| / 127 and its integers rint(127 x / max|row|),
multiplies them with the weight's integers, and puts the two scales, the bias and the epilogue on the sum.  "normed"
takes float32 rows and normalises them (LayerNorm) before that, as every block of the encoder does.  A token score is
the log probability of a given token under a row of logits, with the row's entropy (natural units) and its k likeliest
tokens, ties to the lower index.
"""

import functools
import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-5
BLANK = 0


def listed():
    return [
        # one new row through a small model's up-projection: launch latency and little else
        {"name": "linear-1x1024x512", "op": "linear", "m": 1, "n": 1024, "k": 512, "epi": "bias", "normed": False},
        # one new row through the wide model's up-projection: the weights are read once, nothing is reused
        {"name": "linear-1x16384x4096", "op": "linear", "m": 1, "n": 16384, "k": 4096, "epi": "swish", "normed": False},
        # a command of two seconds: 99 frames into the gated projection
        {"name": "linear-99x2048x1024-glu", "op": "linear", "m": 99, "n": 2048, "k": 1024, "epi": "glu", "normed": False},
        # sizes that are multiples of nothing, float32 out
        {"name": "linear-1237x777x1000-f32", "op": "linear", "m": 1237, "n": 777, "k": 1000, "epi": "float", "normed": False},
        # one utterance of 30 s, down-projection onto the float32 residual stream
        {"name": "linear-1504x1024x4096-residual", "op": "linear", "m": 1504, "n": 1024, "k": 4096, "epi": "residual", "normed": False},
        # the batch of 32 x 30 s, up-projection after its LayerNorm
        {"name": "linear-48128x4096x1024-normed", "op": "linear", "m": 48128, "n": 4096, "k": 1024, "epi": "swish", "normed": True},
        # the same batch, down-projection onto the residual stream
        {"name": "linear-48128x1024x4096-residual", "op": "linear", "m": 48128, "n": 1024, "k": 4096, "epi": "residual", "normed": False},
        # the wide model at batch 8 x 30 s
        {"name": "linear-12032x16384x4096", "op": "linear", "m": 12032, "n": 16384, "k": 4096, "epi": "swish", "normed": False},
        # the benchmark batch's emitted tokens under the framework's own vocabulary
        {"name": "ctc-32x1504x32", "op": "ctc", "batch": 32, "frames": 1504, "vocab": 32, "pitch": 256, "top": 4},
        # one answer of one model with a large vocabulary
        {"name": "scores-1x131072", "op": "scores", "rows": 1, "vocab": 131072, "pitch": 131072, "dtype": "bfloat16", "given": 1, "top": 8, "masked": False},
        # rows of an odd vocabulary that start at any alignment, a third of it ruled out
        {"name": "scores-513x50257-masked", "op": "scores", "rows": 513, "vocab": 50257, "pitch": 50257, "dtype": "float32", "given": 4, "top": 20, "masked": True},
        # scoring a whole batch of texts
        {"name": "scores-8192x32000", "op": "scores", "rows": 8192, "vocab": 32000, "pitch": 32000, "dtype": "bfloat16", "given": 1, "top": 5, "masked": False},
    ]


@functools.lru_cache(maxsize=None)
def _ops():
    """The framework's operators on torch tensors."""
    package = str(Path(__file__).resolve().parent.parent / "omnilingual-asr_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from omnilingual_asr import ops
    return ops


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "scores", "scores", "ctc"])
    if kind == "linear":
        epi = rng.choice(["bias", "swish", "glu", "residual", "float"])
        normed = rng.random() < 0.25
        while True:
            m, n, k = _log_uniform(rng, 1, 48128), _log_uniform(rng, 33, 16384), _log_uniform(rng, 65, 16384)
            if rng.random() < 0.5:
                n, k = (n + 63) // 64 * 64, (k + 63) // 64 * 64
            if normed:
                k = rng.choice([512, 1024, 2048, 4096])
            if epi == "glu":
                n = (n + 31) // 32 * 32
            if m * n * k <= 2 ** 39 and m * max(n, k) <= 2 ** 28:
                return {"op": "linear", "m": m, "n": n, "k": k, "epi": epi, "normed": normed}
    if kind == "scores":
        vocab = _log_uniform(rng, 30, 200000)
        rows = min(_log_uniform(rng, 1, 16384), 2 ** 27 // vocab)
        pitch = vocab + rng.choice([0, 0, rng.randrange(1, 64), -vocab % 256])
        return {"op": "scores", "rows": rows, "vocab": vocab, "pitch": pitch, "dtype": rng.choice(["float32", "bfloat16"]),
                "given": rng.randrange(1, 6), "top": rng.randrange(0, 21), "masked": rng.random() < 0.4}
    return {"op": "ctc", "batch": _log_uniform(rng, 1, 64), "frames": 32 * _log_uniform(rng, 2, 60),
            "vocab": rng.randrange(20, 257), "pitch": 256, "top": rng.randrange(0, 9)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = normal(m, k).mul_(0.25 + 2.0 * uniform(m, 1))      # rows of different sizes
        x[:, :: 97] *= 6.0                                      # and a few channels that stand out, as activations have them
        if case["normed"]:
            state.update(gain=1.0 + 0.1 * normal(k), shift=0.1 * normal(k))
        else:
            x = x.to(torch.bfloat16)
        codes = normal(n, k).mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)
        state.update(x=x, codes=codes, scale=(0.5 + uniform(n)) / (40.0 * math.sqrt(k)), bias=0.5 * normal(n),
                     resid=normal(m, n) if case["epi"] == "residual" else None)
        if own:     # the weight laid out once, as a model keeps it
            state["layer"] = _ops().LinearI8.from_codes(codes, state["scale"], state["bias"])
        return state
    if case["op"] == "ctc":
        b, t, v = case["batch"], case["frames"], case["vocab"]
        lengths = (t * (0.4 + 0.6 * uniform(b))).long().clamp(1, t)
        lengths[0] = t
        logits = normal(b, t, case["pitch"])
        peak = (v * uniform(b, t // 4)).long().clamp(0, v - 1).repeat_interleave(4, dim=1)      # a symbol lasts a few frames
        logits.scatter_add_(2, peak[..., None], 6.0 + 2.0 * normal(b, t, 1))
        logits[..., v:] = -1e30                                   # the columns behind the vocabulary, as the padded head writes them
        ids = logits[..., :v].argmax(dim=2)
        last = torch.cat([torch.full_like(ids[:, :1], -1), ids[:, :-1]], dim=1)
        keep = (ids != BLANK) & (ids != last) & (torch.arange(t, device="cuda") < lengths[:, None])
        place = keep.cumsum(dim=1) - 1
        tokens = torch.full((b, t + 1), -1, dtype=torch.int32, device="cuda")
        frames = torch.full((b, t + 1), -1, dtype=torch.int32, device="cuda")
        at = torch.where(keep, place, torch.full_like(place, t))
        tokens.scatter_(1, at, ids.int())
        frames.scatter_(1, at, torch.arange(t, device="cuda", dtype=torch.int32).expand(b, t).contiguous())
        state.update(logits=logits, tokens=tokens[:, :t].contiguous(), frames=frames[:, :t].contiguous())
        return state
    rows, v = case["rows"], case["vocab"]
    logits = torch.empty(rows * case["pitch"], dtype=getattr(torch, case["dtype"]), device="cuda").view(rows, case["pitch"])
    logits[:, v:] = float("nan")                                  # what lies between the rows is nobody's
    logits = logits[:, :v]
    step = max(1, 2 ** 27 // v)
    for at in range(0, rows, step):
        logits[at: at + step] = (normal(min(step, rows - at), v) * 2.5).to(logits.dtype)
    if case["masked"]:
        for at in range(0, rows, step):
            logits[at: at + step].masked_fill_(uniform(min(step, rows - at), v) < 0.35, -math.inf)
    tokens = (v * uniform(rows, case["given"])).long().clamp(0, v - 1)
    tokens[:, 0] = logits.float().argmax(dim=1) if rows * v <= 2 ** 27 else tokens[:, 0]
    state.update(logits=logits, tokens=tokens.int())
    return state


def _linear(s):
    x = s["x"].float()
    if s["normed"]:
        x = x - x.mean(dim=1, keepdim=True)
        x = x * (x.square().mean(dim=1, keepdim=True) + EPS).rsqrt() * s["gain"] + s["shift"]
    top = x.abs().amax(dim=1, keepdim=True)
    top = torch.where(top > 0, top, torch.full_like(top, 127.0))
    # 64 bits for the quotient: a bf16 value is exactly halfway between two integers often enough (max / 2 is 63.5)
    q = (x.double() * 127.0 / top).round().float()
    y = q @ s["codes"].float().t()
    y = y * (top / 127.0) * s["scale"] + s["bias"]
    if s["epi"] == "swish":
        return (y * torch.sigmoid(y)).to(torch.bfloat16)
    if s["epi"] == "glu":
        y = y.view(y.shape[0], -1, 2, 16)
        return (y[:, :, 0] * torch.sigmoid(y[:, :, 1])).reshape(y.shape[0], -1).to(torch.bfloat16)
    if s["epi"] == "residual":
        return s["resid"] + 0.5 * y
    return y if s["epi"] == "float" else y.to(torch.bfloat16)


def _best(z, k):
    """The k largest of each row and where they are: equal values in order of their place."""
    v = z.shape[1]
    bits = (z + 0.0).view(torch.int32)                              # -0.0 becomes 0.0
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()    # ordered as the values are
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(v, device=z.device))
    ids = 2 ** 32 - 1 - (key.topk(min(k, v), dim=1).values & 0xFFFFFFFF)
    return z.gather(1, ids), ids


def _row_scores(z, k):
    m = z.amax(dim=1, keepdim=True)
    d = z - m
    e = d.exp()
    total = e.sum(dim=1, keepdim=True)
    lse = total.log()
    entropy = lse[:, 0] - (e * d.clamp_min(-1e30)).sum(dim=1) / total[:, 0]
    if k == 0:
        none = z.new_empty((z.shape[0], 0))
        return m, lse, entropy, none.int(), none
    best, ids = _best(z, k)
    ids = torch.where(best == -math.inf, torch.full_like(ids, -1), ids).int()
    best = best - m - lse
    if ids.shape[1] < k:
        pad = (0, k - ids.shape[1])
        ids, best = torch.nn.functional.pad(ids, pad, value=-1), torch.nn.functional.pad(best, pad, value=-math.inf)
    return m, lse, entropy, ids, best


def _scores(s):
    z = s["logits"].float()
    m, lse, entropy, ids, best = _row_scores(z, s["top"])
    return {"logprobs": z.gather(1, s["tokens"].long()) - m - lse, "entropy": entropy, "ids": ids, "best": best}


def _ctc(s):
    tokens, frames = s["tokens"].long(), s["frames"].long()
    b, t = tokens.shape
    there = tokens >= 0
    z = s["logits"][..., : s["vocab"]].gather(1, frames.clamp_min(0)[..., None].expand(b, t, s["vocab"])).reshape(b * t, -1)
    m, lse, entropy, ids, best = _row_scores(z, s["top"])
    logprobs = (z.gather(1, tokens.clamp_min(0).view(-1, 1)) - m - lse).view(b, t)
    zero = torch.zeros((), device=z.device)
    return {"logprobs": torch.where(there, logprobs, zero), "entropy": torch.where(there, entropy.view(b, t), zero),
            "ids": torch.where(there[..., None], ids.view(b, t, -1), torch.full_like(ids, -1).view(b, t, -1)),
            "best": torch.where(there[..., None], best.view(b, t, -1), torch.full_like(best, -math.inf).view(b, t, -1))}


def run(state):
    if own:
        if state["op"] == "linear":
            layer, x = state["layer"], state["x"]
            if state["normed"]:
                return layer.normed(x, state["gain"], state["shift"], eps=EPS, epilogue=state["epi"], resid=state["resid"], alpha=0.5)
            return layer(x, epilogue=state["epi"], resid=state["resid"], alpha=0.5)
        if state["op"] == "ctc":
            r = _ops().ctc_token_scores(state["logits"], state["tokens"], state["frames"], vocab=state["vocab"], alternatives=state["top"])
        else:
            r = _ops().token_scores(state["logits"], state["tokens"], alternatives=state["top"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "ids": r.ids, "best": r.best}
    return {"linear": _linear, "scores": _scores, "ctc": _ctc}[state["op"]](state)


def work(case):
    if case["op"] == "linear":
        m, n, k, epi = case["m"], case["n"], case["k"], case["epi"]
        out = {"bias": 2 * m * n, "swish": 2 * m * n, "glu": m * n, "residual": 8 * m * n, "float": 4 * m * n}[epi]
        return {"bytes": (4 if case["normed"] else 2) * m * k + n * k + 8 * n + out + (8 * k if case["normed"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "ctc":
        rows = case["batch"] * case["frames"]
        # about a frame in four emits a token: its row is read; every place of the outputs is written
        return {"bytes": rows // 4 * case["vocab"] * 4 + rows * (8 + 8 + 8 * case["top"]), "flops": rows // 4 * case["vocab"] * 6}
    rows, size = case["rows"], 4 if case["dtype"] == "float32" else 2
    return {"bytes": rows * (case["vocab"] * size + 8 * case["given"] + 4 + 8 * case["top"]), "flops": rows * case["vocab"] * 6}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        if case["normed"]:
            mean = x.mean(1, keepdim=True)
            x = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS) * s["gain"].double() + s["shift"].double()
        biggest = x.abs().max(dim=1, keepdim=True).values
        biggest = biggest.masked_fill(biggest == 0, 127.0)
        integers = torch.round(127.0 * x / biggest)
        y = torch.matmul(integers, s["codes"].double().T) * biggest / 127.0
        y = y * s["scale"].double()[None, :] + s["bias"].double()[None, :]
        if case["epi"] == "swish":
            return y / (1.0 + torch.exp(-y))
        if case["epi"] == "glu":
            group = y.reshape(y.shape[0], y.shape[1] // 32, 32)
            return (group[:, :, :16] / (1.0 + torch.exp(-group[:, :, 16:]))).reshape(y.shape[0], y.shape[1] // 2)
        return s["resid"].double() + 0.5 * y if case["epi"] == "residual" else y
    if case["op"] == "ctc":
        b, t = s["tokens"].shape
        logp = torch.log_softmax(s["logits"][:, :, : case["vocab"]].double(), dim=2)
        chosen = logp[torch.arange(b, device="cuda")[:, None], s["frames"].long().clamp(min=0)]
        absent = s["tokens"] < 0
        given = chosen.gather(2, s["tokens"].long().clamp(min=0)[..., None])[..., 0].masked_fill(absent, 0.0)
        best = chosen.sort(dim=2, descending=True).values[..., : case["top"]].masked_fill(absent[..., None], -math.inf)
        return {"logprobs": given, "entropy": -(chosen.exp() * chosen).sum(2).masked_fill(absent, 0.0), "ids": None, "best": best}
    rows, v, k = case["rows"], case["vocab"], case["top"]
    given, entropy, best = [], [], []
    step = max(1, 2 ** 26 // v)
    for at in range(0, rows, step):
        logp = torch.log_softmax(s["logits"][at: at + step].double(), dim=1)
        given.append(logp.gather(1, s["tokens"][at: at + step].long()))
        entropy.append(-torch.nan_to_num(logp.exp() * logp, nan=0.0).sum(1))
        part = logp.topk(min(k, v), dim=1).values if k else logp[:, :0]
        best.append(torch.nn.functional.pad(part, (0, k - part.shape[1]), value=-math.inf))
    return {"logprobs": torch.cat(given), "entropy": torch.cat(entropy), "ids": None, "best": torch.cat(best)}
