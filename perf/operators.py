"""The 8-bit integer path of a dense model and the scores of its output tokens, as cases that can be timed.

Three kinds of operators make up that path: a row of activations in 8 bits with a scale (after a normalisation, with the
residual's addition, or after the gated unit), the product of such rows with 8-bit matrices, and the log probabilities of
given tokens with the entropy and the best alternatives.  `run` computes them in their plain form or, with `own`, by this
library's calls.  Shapes are those of the benchmark: a dense 27B-class layer (hidden 5120, attention width 6144, key / value
width 1024, feed-forward 17408), a vocabulary of 151936 and a 2048-wide model with a head over it.
"""
import math

import torch

own = False

EPS = 1e-6
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": F32, "bf16": BF16}
HIDDEN, ATTN, KV, FFN, VOCAB = 5120, 6144, 1024, 17408, 151936


def listed():
    return [
        # The norm between two blocks of a layer, one sequence decoding: what a call costs.
        {"name": "norm_m1", "kind": "norm", "m": 1, "n": HIDDEN, "type": "f32"},
        # The same for a chunk of a prompt, bf16 residual stream.
        {"name": "norm_m2048", "kind": "norm", "m": 2048, "n": HIDDEN, "type": "bf16"},
        # The gated unit before the down projection: a few sequences decoding, and the ragged rest of a prompt.
        {"name": "glu_m7", "kind": "glu", "m": 7, "n": FFN, "type": "f32"},
        {"name": "glu_m1021", "kind": "glu", "m": 1021, "n": FFN, "type": "bf16"},
        # q | k | v of one decoding sequence.
        {"name": "qkv_m1", "kind": "product", "m": 1, "rows": f"{ATTN} {KV} {KV}", "cols": HIDDEN, "type": "f32"},
        # gate | up of sixteen sequences.
        {"name": "gate_up_m16", "kind": "product", "m": 16, "rows": f"{FFN} {FFN}", "cols": HIDDEN, "type": "f32"},
        # The down projection of a short prompt of odd length.
        {"name": "down_m509", "kind": "product", "m": 509, "rows": f"{HIDDEN}", "cols": FFN, "type": "bf16"},
        # gate | up of a full chunk of a prompt.
        {"name": "gate_up_m2048", "kind": "product", "m": 2048, "rows": f"{FFN} {FFN}", "cols": HIDDEN, "type": "bf16"},
        # The scores of one sampled token and its twenty best alternatives.
        {"name": "scores_m1", "kind": "scores", "m": 1, "n": VOCAB, "k": 20, "type": "f32"},
        # A batch of decoding sequences, five alternatives.
        {"name": "scores_m64", "kind": "scores", "m": 64, "n": VOCAB, "k": 5, "type": "f32"},
        # A prompt scored token by token.
        {"name": "scores_m1021", "kind": "scores", "m": 1021, "n": VOCAB, "k": 8, "type": "bf16"},
        # The end of a decode step of four sequences: final norm in 8 bits, output head, scores.
        {"name": "head_m4", "kind": "head", "m": 4, "n": 2048, "rows": f"{VOCAB}", "k": 8, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "glu", "product", "product", "product", "scores", "scores", "head"])
    some = rng.choice(["f32", "bf16"])
    if kind in ("norm", "glu"):
        n = 4 * _log(rng, 32, (8192 if kind == "norm" else FFN) // 4)
        return {"kind": kind, "m": _log(rng, 1, 2048), "n": n, "type": some}
    if kind == "product":
        cols = 16 * _log(rng, 32, FFN // 16)
        many = [_log(rng, 128, FFN) for _ in range(rng.choice([1, 1, 2, 3]))]
        most = min(2048, 2048 * 2 * FFN * HIDDEN // (sum(many) * cols))
        return {"kind": kind, "m": min(most, rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 2048)])), "rows": " ".join(map(str, many)), "cols": cols,
                "type": some}
    n = _log(rng, 2000, VOCAB)
    if kind == "scores":
        return {"kind": kind, "m": _log(rng, 1, 1021), "n": n, "k": rng.choice([0, 1, _log(rng, 2, 32)]), "type": some}
    return {"kind": kind, "m": _log(rng, 1, 32), "n": 16 * _log(rng, 32, 320), "rows": str(n), "k": _log(rng, 1, 32), "type": "f32"}


# ---------------------------------------------------------------- inputs

_device = None


def device():
    """The process's one handle.  It shares the stream that torch works on from then on: one of its own, since a handle takes
    the default stream for its own."""
    global _device
    if _device is None:
        from ferrum_b200 import surface
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.Stream())
        _device = surface.Device(0)
    return _device


def _rows_of(case):
    return [int(r) for r in case["rows"].split()]


def _matrix(gen, rows, cols):
    """A matrix of 8-bit integers and its scale per row: normal weights of deviation 0.02, the largest of a row at 127."""
    q = torch.empty(rows, cols, dtype=torch.int8, device="cuda")
    s = torch.empty(rows, dtype=F32, device="cuda")
    for at in range(0, rows, 8192):
        w = 0.02 * torch.randn(min(8192, rows - at), cols, device="cuda", generator=gen)
        s[at:at + 8192] = w.abs().amax(1) / 127
        q[at:at + 8192] = torch.round(w / s[at:at + 8192, None]).to(torch.int8)
    return q, s


def prepare(case, seed):
    if own:
        device()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 29)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    kind, m, t = case["kind"], case["m"], TYPES[case["type"]]
    s = {"kind": kind, "m": m, "k": case.get("k", 0), "type": t}
    new = lambda *shape, dtype=F32: torch.empty(shape, dtype=dtype, device="cuda")
    if kind in ("norm", "head"):
        n = case["n"]
        # A residual stream has a few channels that are far larger than the rest.
        s["x"] = (randn(m, n) * (1 + 20 * (torch.rand(n, device="cuda", generator=gen) < 0.004))).to(t)
        s["r"], s["w"] = (0.5 * randn(m, n)).to(t), 1 + 0.1 * randn(n)
        s["h"], s["q"], s["s"] = new(m, n, dtype=t), new(m, n, dtype=torch.int8), new(m)
    elif kind == "glu":
        n = case["n"]
        s["gate"], s["up"] = (2 * randn(m, n)).to(t), randn(m, n).to(t)
        s["q"], s["s"] = new(m, n, dtype=torch.int8), new(m)
    if kind in ("product", "head"):
        cols = case["cols"] if kind == "product" else case["n"]
        s["weights"] = [_matrix(gen, r, cols) for r in _rows_of(case)]
        s["y"] = [new(m, r, dtype=t) for r in _rows_of(case)]
        if kind == "product":
            x = randn(m, cols)
            s["xs"] = x.abs().amax(1) / 127
            s["xq"] = torch.round(x / s["xs"][:, None]).to(torch.int8)
        if own:  # a program keeps the library's matrices
            from ferrum_b200 import surface
            s["matrices"] = [surface.Matrix.from_i8(device(), q, scales) for q, scales in s["weights"]]
    if kind == "scores":
        n = case["n"]
        # A model's logits: a wide bulk, a few likely tokens, and in every other row tokens that a grammar forbids.
        l = 2.5 * randn(m, n)
        l.scatter_(1, torch.randint(0, n, (m, 6), device="cuda", generator=gen), 12 + 2 * randn(m, 6))
        forbidden = torch.rand(n, device="cuda", generator=gen) < 0.3
        l[1::2, forbidden] = -math.inf
        s["logits"] = l.to(t)
    if kind in ("scores", "head"):
        n = case["n"] if kind == "scores" else _rows_of(case)[0]
        k = s["k"]
        s["ids"] = torch.randint(0, n, (m,), device="cuda", generator=gen, dtype=torch.int32)
        if kind == "scores":  # most given tokens are likely ones
            s["ids"][::3] = s["logits"][::3].float().argmax(1).to(torch.int32)
        s["logprobs"], s["ranks"], s["entropy"] = new(m), new(m, dtype=torch.int32), new(m)
        s["top"], s["top_ids"] = (new(m, k), new(m, k, dtype=torch.int32)) if k else (None, None)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from ferrum_b200 import surface as S
    d, m, kind = device(), s["m"], s["kind"]
    if kind in ("norm", "head"):
        S.add_rmsnorm_i8(d, s["x"], s["r"], s["w"], EPS, m, s["h"], s["q"], s["s"])
        if kind == "norm":
            return [s["h"], torch.mul(s["q"], s["s"][:, None]), s["s"]]
        S.project_i8(d, s["matrices"][0], s["q"], s["s"], m, s["y"][0])
        _own_scores(S, d, s, s["y"][0])
        return [s["h"], s["y"][0]] + _scores_of(s)
    if kind == "glu":
        S.glu_i8(d, s["gate"], s["up"], m, s["q"], s["s"])
        return [torch.mul(s["q"], s["s"][:, None]), s["s"]]
    if kind == "product":
        if len(s["matrices"]) == 1:
            S.project_i8(d, s["matrices"][0], s["xq"], s["xs"], m, s["y"][0])
        else:
            S.project_many_i8(d, s["matrices"], s["xq"], s["xs"], m, s["y"])
        return s["y"]
    _own_scores(S, d, s, s["logits"])
    return _scores_of(s)


def _own_scores(S, d, s, logits):
    S.token_logprobs(d, logits, logits.shape[1], s["m"], s["ids"], s["logprobs"], s["ranks"], s["entropy"], s["k"], s["top"], s["top_ids"])


def _scores_of(s):
    return [s["logprobs"], s["ranks"], s["entropy"]] + ([s["top"], s["top_ids"]] if s["k"] else [])


def _to_8_bits(v, factor):
    """Rows of 64-bit values as whole numbers up to 127 of each row's largest (64 bits: a value next to the border of two
    whole numbers has to fall on the right side), and what one of them stands for."""
    most = v.abs().amax(1, keepdim=True)
    q = torch.round(v * 127 / torch.where(most > 0, most, 1.0))
    return q, (most * factor / 127).to(F32)


def _run_plain(s):
    kind, t = s["kind"], s["type"]
    if kind in ("norm", "head"):
        h = (s["x"].float() + s["r"].float()).to(t)
        h64 = h.double()
        q, scale = _to_8_bits(h64 * s["w"].double(), 1 / torch.sqrt(h64.square().mean(1, keepdim=True) + EPS))
        if kind == "norm":
            return [h, q.float() * scale, scale[:, 0]]
        wq, ws = s["weights"][0]
        # Whole numbers past 2^24, and their order decides ranks: 64 bits.
        logits = (q @ wq.double().T).float() * scale * ws
        return [h, logits] + _plain_scores(logits, s["ids"], s["k"])
    if kind == "glu":
        g, u = s["gate"].double(), s["up"].double()
        q, scale = _to_8_bits(g / (1 + torch.exp(-g)) * u, 1.0)
        return [q.float() * scale, scale[:, 0]]
    if kind == "product":
        x = s["xq"].float()
        return [((x @ wq.float().T) * s["xs"][:, None] * ws).to(t) for wq, ws in s["weights"]]
    return _plain_scores(s["logits"].float(), s["ids"], s["k"])


def _plain_scores(l, ids, k):
    m, n = l.shape
    at = l.amax(1, keepdim=True)
    e = torch.exp(l - at)
    total = e.sum(1, keepdim=True)
    z = at + torch.log(total)
    given = l.gather(1, ids.long()[:, None])
    ranks = 1 + (l > given).sum(1, dtype=torch.int32)
    p = e / total
    entropy = -torch.where(p > 0, p * (l - z), 0.0).sum(1)
    out = [(given - z)[:, 0], ranks, entropy]
    if k:
        # The largest k by value, ties to the lower index: one whole number for both.
        bits = (l + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 2 ** 32 + torch.arange(n - 1, -1, -1, device=l.device)
        top = n - 1 - (order.topk(k, 1).values & 0xFFFFFFFF)
        out += [l.gather(1, top) - z, top.to(torch.int32)]
    return out


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind, m = s["kind"], s["m"]
    if kind == "product":
        x = s["xq"].double().mul(s["xs"].double().unsqueeze(1))
        return [torch.einsum("tk,ok->to", x, wq.double()).mul(ws.double()) for wq, ws in s["weights"]]
    if kind == "glu":
        v = torch.sigmoid(s["gate"].double()).mul(s["gate"].double()).mul(s["up"].double())
        step = v.abs().max(dim=1, keepdim=True).values.div(127.0)
        return [torch.round(v / step).mul(step), step.squeeze(1)]
    if kind == "scores":
        return _exact_scores(s["logits"].double(), s)
    h = torch.add(s["x"], s["r"]).double()  # the sum as it is kept
    v = h.mul(s["w"].double())
    rms = h.pow(2).sum(dim=1, keepdim=True).div(h.shape[1]).add(EPS).pow(0.5)
    step = v.abs().max(dim=1, keepdim=True).values.div(127.0)
    values = torch.round(v / step).mul(step).div(rms)
    if kind == "norm":
        return [h, values, step.div(rms).squeeze(1)]
    wq, ws = s["weights"][0]
    logits = torch.einsum("tk,ok->to", values, wq.double()).mul(ws.double())
    return [h, logits] + _exact_scores(logits, s)


def _exact_scores(l, s):
    logs = torch.log_softmax(l, dim=1)
    entropy = torch.special.entr(logs.exp()).sum(dim=1)
    out = [logs[torch.arange(s["m"], device=l.device), s["ids"].long()], None, entropy]
    return out + ([logs.sort(dim=1, descending=True).values[:, :s["k"]], None] if s["k"] else [])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind, m, size = case["kind"], case["m"], 2 if case["type"] == "bf16" else 4
    norm = lambda n: {"bytes": m * n * (3 * size + 1) + 4 * n + 4 * m, "flops": 8 * m * n}
    scores = lambda n, logits: {"bytes": logits + m * (16 + 8 * case["k"]), "flops": 6 * m * n}
    product = lambda rows, cols: {"bytes": rows * cols + 4 * rows + m * (cols + 4) + m * rows * size, "flops": 2 * m * rows * cols}
    if kind == "norm":
        return norm(case["n"])
    if kind == "glu":
        return {"bytes": m * case["n"] * (2 * size + 1) + 4 * m, "flops": 10 * m * case["n"]}
    if kind == "scores":
        return scores(case["n"], m * case["n"] * size)
    rows = sum(_rows_of(case))
    if kind == "product":
        return product(rows, case["cols"])
    parts = [norm(case["n"]), product(rows, case["n"]), scores(rows, m * rows * size)]
    return {w: sum(p[w] for p in parts) for w in ("bytes", "flops")}
