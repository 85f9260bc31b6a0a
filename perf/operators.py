"""The work a program hands to this library's 8-bit integer passes and to its verification of drafted tokens, as measurable cases.

  op        what is called                                                        stands for
  rows_i8   Runtime.rows_i8: rows normalised (after the residual's addition) or   the activations of a pass's projections, in 8 bits with a
            gated (silu(x) * x2), as 8-bit integers with a scale per row          scale per token
  qmm_i8    Runtime.qmm_i8: 8-bit activations times an 8-bit weight tensor        projections of a decode step, a verification pass, a prompt
  verify    Runtime.verify: drafted tokens against the target's probabilities     the end of a speculative decoding step

`run` computes them in elementary torch operations where `own` is false, and calls the library where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16}
EPS = 1e-6
MOST_BYTES = 3.5e8    # a drawn case's inputs and outputs, at most
MOST_MACS = 4096 * 17408 * 5120


def listed():
    return [
        # One decode step's row of hidden values: residual, norm, 8 bits.  Latency.
        {"name": "norm_1", "op": "rows_i8", "ntok": 1, "cols": 5120, "type": "fp32", "residual": True, "norm": True, "gated": False},
        # A verification pass of four rows: silu(gate) * up for the down projection.
        {"name": "gated_4", "op": "rows_i8", "ntok": 4, "cols": 17408, "type": "fp32", "residual": False, "norm": False, "gated": True},
        # A prompt pass, residual rows in 16 bits, a number of rows that is no multiple of anything.
        {"name": "norm_prompt", "op": "rows_i8", "ntok": 4001, "cols": 5120, "type": "fp16", "residual": True, "norm": True, "gated": False},
        # The gate projection of a decode step: one pass over the weights.
        {"name": "i8_1", "op": "qmm_i8", "ntok": 1, "rows": 17408, "cols": 5120, "type": "fp32"},
        # A small projection of a verification pass: hardly anything to read.
        {"name": "i8_4_small", "op": "qmm_i8", "ntok": 4, "rows": 1024, "cols": 5120, "type": "fp32"},
        # The down projection of a batch's verification passes.
        {"name": "i8_24_down", "op": "qmm_i8", "ntok": 24, "rows": 5120, "cols": 17408, "type": "fp32"},
        # Odd sizes everywhere.
        {"name": "i8_odd", "op": "qmm_i8", "ntok": 77, "rows": 1001, "cols": 4999, "type": "fp16"},
        # A prompt's chunk.
        {"name": "i8_512", "op": "qmm_i8", "ntok": 512, "rows": 17408, "cols": 5120, "type": "fp32"},
        # A long prompt, outputs in 16 bits.
        {"name": "i8_4096", "op": "qmm_i8", "ntok": 4096, "rows": 17408, "cols": 5120, "type": "fp16"},
        # One sequence with three drafts, the default depth of a drafter.
        {"name": "verify_1", "op": "verify", "seqs": 1, "drafts": 3, "vocab": 151936, "type": "fp32", "draft": "logits", "ragged": False},
        # Drafts that a lookup proposed (no probabilities of their own), a padded batch, an odd vocabulary.
        {"name": "verify_lookup", "op": "verify", "seqs": 13, "drafts": 7, "vocab": 32003, "type": "fp32", "draft": "tokens", "ragged": True},
        # A full server.
        {"name": "verify_64", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 151936, "type": "fp32", "draft": "logits", "ragged": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rows_i8", "qmm_i8", "qmm_i8", "verify"])
    kind = rng.choice(["fp32", "fp32", "fp16"])
    while True:
        if op == "rows_i8":
            gated = rng.random() < 0.35
            norm = not gated or rng.random() < 0.3
            case = {"op": op, "ntok": _log(rng, 1, 4096), "cols": _log(rng, 33, 20480), "type": kind, "residual": not gated and rng.random() < 0.7,
                    "norm": norm, "gated": gated}
        elif op == "qmm_i8":
            case = {"op": op, "ntok": _log(rng, 1, 4096), "rows": _log(rng, 17, 40000), "cols": _log(rng, 33, 20480), "type": kind}
            if case["ntok"] * case["rows"] * case["cols"] > MOST_MACS:
                continue
        else:
            case = {"op": op, "seqs": _log(rng, 1, 64), "drafts": rng.randint(0, 8), "vocab": _log(rng, 101, 152064), "type": kind,
                    "draft": rng.choice(["logits", "logits", "tokens"]), "ragged": rng.random() < 0.5}
        if work(case)["bytes"] <= MOST_BYTES:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


class _State:
    """A pass's tensors, and where the library runs it the runtime that knows them by name."""

    def __init__(self, case, seed):
        self.case = case
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.t = {}
        self.rt = None
        if own:
            from vinf_3080ti_b200.runtime import Runtime

            self.rt = Runtime()

    def buffer(self, name, tensor):
        self.t[name] = tensor
        if self.rt is not None:
            self.rt.bind(name, tensor.data_ptr(), tensor.numel(), tensor.element_size())
        return tensor

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def uniform(self, low, high, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda") * (high - low) + low


def _pitch(cols):
    return (cols + 15) // 16 * 16


def _bytes_of(values, pitch):
    """Whole numbers as 8-bit rows of `pitch` bytes, zeros behind the last."""
    rows, cols = values.shape
    out = torch.zeros((rows, pitch), dtype=torch.int8, device="cuda")
    out[:, :cols] = values
    return out


def prepare(case, seed):
    s = _State(case, seed)
    if case["op"] == "rows_i8":
        m, n, kind = case["ntok"], case["cols"], TYPES[case["type"]]
        channels = torch.where(s.uniform(0, 1, n) < 0.002, 20.0, 1.0)  # a few columns are much larger, as in hidden states
        s.buffer("x", (s.normal(m, n) * channels).to(kind))
        if case["gated"]:
            s.buffer("x2", s.normal(m, n).to(kind))
        if case["residual"]:
            s.buffer("residual", (s.normal(m, n) * 3 * channels).to(kind))
            s.buffer("sum", torch.zeros((m, n), dtype=kind, device="cuda"))
        if case["norm"]:
            s.buffer("gain", s.uniform(0.5, 1.5, n))
        s.buffer("q", torch.zeros((m, _pitch(n)), dtype=torch.int8, device="cuda"))
        s.buffer("scale", torch.zeros(m, device="cuda"))
    elif case["op"] == "qmm_i8":
        m, rows, cols, kind = case["ntok"], case["rows"], case["cols"], TYPES[case["type"]]
        w = _bytes_of((s.normal(rows, cols) * 30).round().clamp(-127, 127), _pitch(cols))
        w_scale = s.uniform(1e-4, 1e-3, rows)
        s.t["w"], s.t["w_scale"] = w, w_scale
        if s.rt is not None:
            s.rt.bind_i8("w", w.data_ptr(), w_scale.data_ptr(), cols, rows)
        s.buffer("q", _bytes_of((s.normal(m, cols) * 30).round().clamp(-127, 127), _pitch(cols)))
        s.buffer("scale", s.uniform(1e-3, 1e-1, m))
        s.buffer("y", torch.zeros((m, rows), dtype=kind, device="cuda"))
    else:
        n, k, vocab, kind = case["seqs"], case["drafts"], case["vocab"], TYPES[case["type"]]
        target = s.normal(n, k + 1, vocab) * 3
        temperature = s.uniform(0.5, 1.2, n)
        if n > 3:
            temperature[3] = 0.0  # a greedy sequence among the others
        if case["draft"] == "logits" and k > 0:
            draft = s.buffer("draft", (target[:, :k] + 0.7 * s.normal(n, k, vocab)).to(kind))
        else:
            draft = target[:, :k] + 0.7 * s.normal(n, k, vocab)
        s.buffer("target", target.to(kind))
        at = temperature.clamp_min(1e-3)[:, None, None]
        gumbel = -torch.log(-torch.log(s.uniform(0, 1, n, k, vocab).clamp(1e-20, 1 - 2**-24))) if k > 0 else draft
        s.buffer("tokens", (draft.float() / at + gumbel).argmax(-1).int() if k > 0 else torch.zeros((n, 1), dtype=torch.int32, device="cuda"))
        del target, draft, gumbel
        s.buffer("uniforms", torch.rand((n, k + 1), generator=s.gen, device="cuda"))
        s.buffer("temperature", temperature)
        if case["ragged"]:
            s.buffer("lens", torch.randint(0, k + 1, (n,), generator=s.gen, device="cuda", dtype=torch.int32))
        s.buffer("out", torch.zeros((n, k + 2), dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    return s


# ---- passes ---------------------------------------------------------------------------------------------------------


def _rows_i8(case, t):
    x = t["x"]
    total = None
    v = x.double()
    if case["gated"]:
        v = v / (1 + torch.exp(-v)) * t["x2"].double()
    if case["residual"]:
        total = (x.float() + t["residual"].float()).to(x.dtype)
        v = total.double()
    if case["norm"]:
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * t["gain"].double()
    # 64 bits: which of two whole numbers a value is rounded to does not hang on how 32 bits got there
    scale = (v.abs().amax(-1) / 127).float()
    q = torch.where(scale[:, None] > 0, torch.round(v / scale.double()[:, None]), 0.0).clamp(-127, 127).to(torch.int8)
    return {"q": q, "scale": scale, "sum": total}


def _qmm_i8(case, t):
    cols = case["cols"]
    sums = t["q"][:, :cols].float() @ t["w"][:, :cols].float().T
    return {"y": (sums * t["scale"][:, None] * t["w_scale"]).to(TYPES[case["type"]])}


def _weights(logits, temperature):
    """exp(l / T) over the row's largest; T = 0: one at the lowest index of the largest."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    at = temperature.double()[:, None, None]
    index = torch.arange(x.shape[-1], device=x.device)
    first = torch.where(x == top, index, x.shape[-1]).amin(-1, keepdim=True)
    w = torch.where(at > 0, torch.exp((x - top) / torch.where(at > 0, at, 1.0)), (index == first).double())
    return w / w.sum(-1, keepdim=True)


def _verify(case, t):
    n, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    tokens = t["tokens"][:, :k].long()
    p = _weights(t["target"], t["temperature"])
    place = torch.arange(k, device=p.device)
    lens = t["lens"].long() if case["ragged"] else torch.full((n,), k, device=p.device)
    if case["draft"] == "logits" and k > 0:
        q = _weights(t["draft"], t["temperature"])
    else:
        q = (torch.arange(vocab, device=p.device) == tokens[:, :, None]).double()
    u = t["uniforms"].double()
    taken = u[:, :k] * q.gather(2, tokens[:, :, None])[..., 0] < p[:, :k].gather(2, tokens[:, :, None])[..., 0]
    count = (taken & (place < lens[:, None])).long().cumprod(1).sum(1)
    seq = torch.arange(n, device=p.device)
    p_row = p[seq, count]
    q_row = torch.cat([q, torch.zeros_like(p[:, :1])], 1)[seq, count] * (count < lens)[:, None]
    rest = (p_row - q_row).clamp_min(0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p_row)
    sums = rest.cumsum(-1)
    chosen = (sums <= u[:, k:] * sums[:, -1:]).sum(-1)
    out = torch.full((n, k + 2), -1, dtype=torch.int32, device=p.device)
    out[:, 0] = count.int()
    out[:, 1:k + 1] = torch.where(place < count[:, None], tokens, -1).int()
    out.scatter_(1, count[:, None] + 1, chosen[:, None].int())
    return out


def run(s):
    case, rt = s.case, s.rt
    op = case["op"]
    if not own:
        return _rows_i8(case, s.t) if op == "rows_i8" else _qmm_i8(case, s.t) if op == "qmm_i8" else _verify(case, s.t)
    if op == "rows_i8":
        rt.rows_i8("x", "q", "scale", case["cols"], case["ntok"], residual="residual" if case["residual"] else None,
                   total="sum" if case["residual"] else None, norm="gain" if case["norm"] else None, eps=EPS, silu_mul="x2" if case["gated"] else None)
        return {"q": s.t["q"][:, :case["cols"]], "scale": s.t["scale"], "sum": s.t.get("sum")}
    if op == "qmm_i8":
        rt.qmm_i8("w", "q", "scale", "y", case["ntok"])
        return {"y": s.t["y"]}
    rt.verify("target", "draft" if "draft" in s.t else None, "tokens", "uniforms", case["vocab"], case["seqs"], case["drafts"],
              lens="lens" if case["ragged"] else None, temperature="temperature", out="out", blocking=False)
    return s.t["out"]


# ---- what a pass cannot do without, and what it gives in 64 bits -----------------------------------------------------


def work(case):
    elem = 2 if case["type"] == "fp16" else 4
    if case["op"] == "rows_i8":
        values = case["ntok"] * case["cols"]
        read = values * elem * (1 + case["residual"] + case["gated"]) + 4 * case["cols"] * case["norm"]
        return {"bytes": read + values * (1 + elem * case["residual"]) + 4 * case["ntok"], "flops": values * (4 + 4 * case["norm"] + 5 * case["gated"])}
    if case["op"] == "qmm_i8":
        m, rows, cols = case["ntok"], case["rows"], case["cols"]
        return {"bytes": rows * cols + m * cols + 4 * (rows + m) + m * rows * elem, "flops": 2 * m * rows * cols}
    n, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    values = n * vocab * (k + 1 + (k if case["draft"] == "logits" else 0))
    return {"bytes": values * elem + 4 * n * (k + k + 1 + 2 + k + 2), "flops": 3 * values}


def exact(case, seed):
    t = prepare(case, seed).t

    def rows_in_64(case, t):
        x = t["x"].to(torch.float64)
        out = {"q": [], "scale": [], "sum": []}
        for r in range(0, case["ntok"], 512):  # a few rows at a time
            v = x[r:r + 512].clone()
            if case["gated"]:
                v = v * torch.sigmoid(v) * t["x2"][r:r + 512].to(torch.float64)
            if case["residual"]:
                v = torch.add(v, t["residual"][r:r + 512].to(torch.float64)).to(t["x"].dtype).to(torch.float64)
                out["sum"].append(v.clone())
            if case["norm"]:
                norm = torch.linalg.vector_norm(v, dim=1) / math.sqrt(case["cols"])
                v = v / torch.sqrt(norm * norm + EPS)[:, None] * t["gain"].to(torch.float64)
            largest = torch.maximum(v.max(1).values, -v.min(1).values)
            held = (largest / 127).to(torch.float32).to(torch.float64)
            out["q"].append(torch.nan_to_num(v / held[:, None]).round().clamp(-127, 127).to(torch.int8))
            out["scale"].append(largest / 127)
        return {name: torch.cat(parts) if parts else None for name, parts in out.items()}

    def verify_in_64(case, t):
        n, k, vocab = case["seqs"], case["drafts"], case["vocab"]
        host = {name: v.cpu() for name, v in t.items() if name in ("tokens", "uniforms", "temperature", "lens")}

        def spread(row, at):
            row = row.to(torch.float64)
            if at <= 0:
                only = torch.zeros_like(row)
                only[int((row == row.max()).nonzero()[0])] = 1.0
                return only
            return torch.softmax(row / at, 0)

        out = torch.full((n, k + 2), -1, dtype=torch.int32)
        for i in range(n):
            at, drafts = float(host["temperature"][i]), int(host["lens"][i]) if case["ragged"] else k
            j, rest = 0, None
            while j < drafts:
                p, token = spread(t["target"][i, j], at), int(host["tokens"][i, j])
                if "draft" in t:
                    q = spread(t["draft"][i, j], at)
                else:
                    q = torch.zeros_like(p)
                    q[token] = 1.0
                if not float(host["uniforms"][i, j]) * float(q[token]) < float(p[token]):
                    rest = torch.relu(p - q)
                    if float(rest.sum()) == 0:
                        rest = p
                    break
                out[i, 1 + j] = token
                j += 1
            if rest is None:
                rest = spread(t["target"][i, j], at)
            sums = torch.cumsum(rest, 0)
            point = float(host["uniforms"][i, k]) * float(sums[-1])
            out[i, 0] = j
            out[i, 1 + j] = int(torch.searchsorted(sums, torch.tensor([point], dtype=torch.float64, device=sums.device), right=True)[0])
        return out

    if case["op"] == "rows_i8":
        return rows_in_64(case, t)
    if case["op"] == "verify":
        return verify_in_64(case, t)
    m, cols, parts = case["ntok"], case["cols"], []
    for r in range(0, case["rows"], 4096):  # a few weight rows at a time
        w = t["w"][r:r + 4096, :cols].to(torch.float64) * t["w_scale"][r:r + 4096, None].to(torch.float64)
        parts.append((t["q"][:, :cols].to(torch.float64) * t["scale"][:, None].to(torch.float64)) @ w.T)
    return {"y": torch.cat(parts, 1) if parts else torch.zeros((m, 0))}
