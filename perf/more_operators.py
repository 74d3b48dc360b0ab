"""Workloads of the operators around a sequence model's training step and its
token by token use: a gated linear recurrence, dropout on the way to the
residual stream, and the loss against a vocabulary.

Three operators, each in the directions a user calls it:

``rec``   gated linear recurrence along the sequence, gates from their logits
``drop``  dropout from a counter-based generator, added onto a residual
``ce``    softmax cross entropy of hidden rows against a vocabulary matrix

``mode`` is "forward", "train" (forward and gradients) or "step" (one token of
every sequence of a batch, on kept state). ``run`` computes them in plain torch
operations in 32 bits (the recurrence in 64), or, where ``own`` is true, through
``ferrum_gpu.sequence``.
"""

import math
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One token of one conversation: the smallest call, all latency.
        dict(name="rec_step_1", op="rec", mode="step", dtype="bf16", batch=1, length=1,
             channels=2048, ragged=False),
        # One token of a full serving batch.
        dict(name="rec_step_256", op="rec", mode="step", dtype="f16", batch=256, length=1,
             channels=4096, ragged=False),
        # One long prompt: few rows, a long axis.
        dict(name="rec_prompt", op="rec", mode="forward", dtype="bf16", batch=1, length=8191,
             channels=2048, ragged=False),
        # A batch of prompts of different lengths, odd sizes, full precision, trained on.
        dict(name="rec_ragged", op="rec", mode="train", dtype="f32", batch=13, length=777,
             channels=1000, ragged=True),
        # The training step's recurrence.
        dict(name="rec_train", op="rec", mode="train", dtype="bf16", batch=8, length=2048,
             channels=4096, ragged=False),
        # Dropout of one short sequence, an odd number of rows.
        dict(name="drop_short", op="drop", mode="forward", dtype="f16", rows=129, channels=1000,
             p=0.1, residual="f16"),
        # Dropout in training, onto a 32-bit residual stream.
        dict(name="drop_train", op="drop", mode="train", dtype="bf16", rows=16384, channels=2048,
             p=0.1, residual="f32"),
        # The log-likelihoods of a few tokens: bound by reading the vocabulary matrix.
        dict(name="ce_score", op="ce", mode="forward", dtype="bf16", tokens=8, width=2048,
             vocab=32000, masked=0.0, lse_grad=False),
        # A fine-tuning batch of which half the tokens carry no loss, odd sizes.
        dict(name="ce_odd", op="ce", mode="train", dtype="f16", tokens=777, width=999,
             vocab=30011, masked=0.5, lse_grad=False),
        # A small model in full precision, with a penalty on the normaliser.
        dict(name="ce_full", op="ce", mode="train", dtype="f32", tokens=500, width=384,
             vocab=5003, masked=0.0, lse_grad=True),
        # The evaluation loss of one batch.
        dict(name="ce_eval", op="ce", mode="forward", dtype="bf16", tokens=4096, width=2048,
             vocab=32768, masked=0.0, lse_grad=False),
        # The training step's loss: the largest work.
        dict(name="ce_train", op="ce", mode="train", dtype="bf16", tokens=8192, width=2048,
             vocab=32768, masked=0.05, lse_grad=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rec", "rec", "drop", "ce", "ce"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "rec":
        mode = rng.choice(["forward", "train", "step"])
        channels = _log_int(rng, 64, 5000)
        batch = _log_int(rng, 1, 256 if mode == "step" else 16)
        limit = 60_000_000 // (channels * batch)
        length = 1 if mode == "step" else _log_int(rng, 1, max(1, min(8192, limit)))
        return dict(op=op, mode=mode, dtype=dtype, batch=batch, length=length, channels=channels,
                    ragged=mode != "step" and rng.random() < 0.3)
    if op == "drop":
        mode = rng.choice(["forward", "train"])
        channels = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, max(1, min(32768, 30_000_000 // channels)))
        return dict(op=op, mode=mode, dtype=dtype, rows=rows, channels=channels,
                    p=rng.choice([0.05, 0.1, 0.1, 0.2, 0.5]),
                    residual=rng.choice(["", dtype, "f32"]))
    mode = rng.choice(["forward", "train"])
    width = _log_int(rng, 64, 4096)
    vocab = _log_int(rng, 256, 131072)
    cap = 10_000_000_000 if dtype == "f32" else 400_000_000_000
    tokens = _log_int(rng, 1, max(1, min(16384, cap // (width * vocab), 500_000_000 // vocab)))
    return dict(op=op, mode=mode, dtype=dtype, tokens=tokens, width=width, vocab=vocab,
                masked=rng.choice([0.0, 0.05, 0.5]), lse_grad=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs

class _Rand:
    """Seeded random tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std + mean).to(dtype)

    def uniform(self, shape, lo, hi):
        return torch.rand(shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def integers(self, shape, n):
        return torch.randint(n, shape, generator=self.g, device="cuda")


def _lengths(case, r):
    if not case.get("ragged"):
        return None
    b, n = case["batch"], case["length"]
    out = torch.floor(r.uniform((b,), 0, n + 1)).to(torch.int32).clamp_(0, n)
    out[0] = n                       # one sequence fills the batch's length,
    if b > 2:
        out[b // 2] = 0              # one is empty
    return out


def prepare(case, seed):
    r = _Rand(seed)
    dt = _DTYPES[case["dtype"]]
    op, mode = case["op"], case["mode"]
    s = {"case": case}
    if op == "rec":
        b, n, d = case["batch"], case["length"], case["channels"]
        lead = (b, d) if mode == "step" else (b, n, d)
        s["lengths"] = _lengths(case, r)
        s["x"] = r.normal(lead, dt)
        s["ig"] = r.normal(lead, dt)
        s["rg"] = r.normal(lead, dt)
        # memories from a few steps to about a thousand, where the gate is half open
        s["decay"] = -2.0 * torch.log(r.uniform((d,), 0.8, 0.999))
        s["state"] = r.normal((b, d))
        if mode == "train":
            s["dout"] = r.normal(lead, dt)
        if mode == "step":
            s["next_state"] = torch.empty_like(s["state"])
    elif op == "drop":
        m, d = case["rows"], case["channels"]
        s["x"] = r.normal((m, d), dt)
        s["residual"] = r.normal((m, d), _DTYPES[case["residual"]], 2.0) if case["residual"] else None
        s["seed"] = r.integers((1,), 2 ** 62)
        if mode == "train":
            s["dy"] = r.normal((m, d), _DTYPES[case["residual"] or case["dtype"]])
    else:
        t, d, v = case["tokens"], case["width"], case["vocab"]
        s["x"] = r.normal((t, d), dt)
        s["weight"] = r.normal((v, d), dt, 1.5 / math.sqrt(d))
        targets = r.integers((t,), v)
        lost = r.uniform((t,), 0, 1) < case["masked"]
        s["targets"] = torch.where(lost, torch.full_like(targets, -100), targets)
        if mode == "train":
            # the mean over the tokens that count, times the loss scale that
            # training in 16-bit floats of a small range needs
            scale = 1024.0 if case["dtype"] == "f16" else 1.0
            count = (~lost).sum().clamp(min=1)
            s["dloss"] = torch.full((t,), scale, device="cuda") / count
            s["dlse"] = r.normal((t,), std=0.01, mean=0.02) * s["dloss"] if case["lse_grad"] else None
    if own:
        _sequence()
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    which = _OWN if own else _PLAIN
    return which[(case["op"], case["mode"])](state, case)


def _sequence():
    if "ferrum-gpu_b200" not in sys.path:
        sys.path.insert(0, "ferrum-gpu_b200")
    from ferrum_gpu import sequence

    return sequence


# The framework's calls.

def _own_rec_forward(s, c):
    r = _sequence().gated_recurrence(s["x"], s["ig"], s["rg"], s["decay"],
                                     initial_state=s["state"], lengths=s["lengths"])
    return {"out": r.out, "state": r.final_state}


def _own_rec_train(s, c):
    seq = _sequence()
    r = seq.gated_recurrence(s["x"], s["ig"], s["rg"], s["decay"], initial_state=s["state"],
                             lengths=s["lengths"], save_states=True)
    g = seq.gated_recurrence_backward(s["dout"], s["x"], s["ig"], s["rg"], s["decay"], r.states,
                                      lengths=s["lengths"])
    return {"out": r.out, "state": r.final_state, "dx": g.dx, "dig": g.dinput_gate,
            "drg": g.drecurrence_gate, "ddecay": g.ddecay, "dstate": g.dinitial_state}


def _own_rec_step(s, c):
    y = _sequence().gated_recurrence_step(s["x"], s["ig"], s["rg"], s["decay"], s["state"],
                                          next_state=s["next_state"])
    return {"out": y, "state": s["next_state"]}


def _own_drop_forward(s, c):
    return {"y": _sequence().dropout(s["x"], c["p"], s["seed"], residual=s["residual"])}


def _own_drop_train(s, c):
    seq = _sequence()
    y = seq.dropout(s["x"], c["p"], s["seed"], residual=s["residual"])
    return {"y": y, "dx": seq.dropout_backward(s["dy"], c["p"], s["seed"], dtype=s["x"].dtype)}


def _own_ce_forward(s, c):
    r = _sequence().linear_cross_entropy(s["x"], s["weight"], s["targets"])
    return {"loss": r.loss, "lse": r.lse}


def _own_ce_train(s, c):
    seq = _sequence()
    r = seq.linear_cross_entropy(s["x"], s["weight"], s["targets"])
    g = seq.linear_cross_entropy_backward(s["dloss"], s["x"], s["weight"], s["targets"], r.lse,
                                          dlse=s["dlse"])
    return {"loss": r.loss, "lse": r.lse, "dx": g.dx, "dweight": g.dweight}


_OWN = {("rec", "forward"): _own_rec_forward, ("rec", "train"): _own_rec_train,
        ("rec", "step"): _own_rec_step, ("drop", "forward"): _own_drop_forward,
        ("drop", "train"): _own_drop_train, ("ce", "forward"): _own_ce_forward,
        ("ce", "train"): _own_ce_train}


# The plain forms.

def _inside(s, c):
    """Which steps lie inside their sequence, (batch, length, 1)."""
    steps = torch.arange(c["length"], device="cuda")
    return (steps[None] < s["lengths"][:, None])[:, :, None]


def _factors(s):
    """Gates, x, a and sqrt(1 - a^2), in 64 bits: over a memory of a thousand
    steps the rounding of a to 32 bits alone puts the gradient of decay, a sum
    that cancels, off by 1e-5."""
    r = torch.sigmoid(s["rg"].double())
    i = torch.sigmoid(s["ig"].double())
    x = s["x"].double()
    la = -s["decay"].double() * r
    a = torch.exp(la)
    root = torch.sqrt(-torch.expm1(2 * la))
    return r, i, x, a, root


def _plain_states(s, c):
    r, i, x, a, root = _factors(s)
    b = root * i * x
    if s["lengths"] is not None:
        keep = _inside(s, c)
        a = torch.where(keep, a, torch.ones_like(a))
        b = torch.where(keep, b, torch.zeros_like(b))
    states = torch.empty((c["batch"], c["length"] + 1, c["channels"]), dtype=torch.float64,
                         device="cuda")
    states[:, 0] = s["state"]
    for t in range(c["length"]):
        states[:, t + 1] = a[:, t] * states[:, t] + b[:, t]
    return r, i, x, a, root, states


def _shown(states, s, c):
    out = states[:, 1:]
    if s["lengths"] is not None:
        out = torch.where(_inside(s, c), out, torch.zeros_like(out))
    return out.to(s["x"].dtype)


def _plain_rec_forward(s, c):
    states = _plain_states(s, c)[-1]
    return {"out": _shown(states, s, c), "state": states[:, -1].float()}


def _plain_rec_train(s, c):
    r, i, x, a, root, states = _plain_states(s, c)
    dout = s["dout"].double()
    if s["lengths"] is not None:
        dout = torch.where(_inside(s, c), dout, torch.zeros_like(dout))
    grad = torch.empty_like(dout)                 # of the states
    later = torch.zeros_like(states[:, 0])
    for t in range(c["length"] - 1, -1, -1):
        grad[:, t] = dout[:, t] + later
        later = a[:, t] * grad[:, t]
    slope = torch.where(root > 0, a * a / root, torch.zeros_like(root))
    dla = grad * (a * states[:, :-1] - slope * i * x)
    dx, dig = grad * root * i, grad * root * x * i * (1 - i)
    drg = -dla * s["decay"] * r * (1 - r)
    drop = -r * dla
    if s["lengths"] is not None:
        keep = _inside(s, c)
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        dx, dig, drg, drop = (torch.where(keep, v, zero) for v in (dx, dig, drg, drop))
    dt = s["x"].dtype
    return {"out": _shown(states, s, c), "state": states[:, -1].float(), "dx": dx.to(dt),
            "dig": dig.to(dt), "drg": drg.to(dt), "ddecay": drop.sum((0, 1)).float(),
            "dstate": later.float()}


def _plain_rec_step(s, c):
    r, i, x, a, root = _factors(s)
    h = a * s["state"] + root * i * x
    return {"out": h.to(s["x"].dtype), "state": h.float()}


# Philox4x32-10 (J. K. Salmon et al., "Parallel random numbers: as easy as 1, 2,
# 3", SC 2011) on 32-bit words kept in 64-bit integers: the counter is the
# group of four elements and an offset of zero, the key the seed.

def _philox(groups, seed):
    low = 0xFFFFFFFF
    c0, c1 = groups & low, (groups >> 32) & low
    c2, c3 = torch.zeros_like(groups), torch.zeros_like(groups)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57     # their 64 bits, as signed ones
        c0, c1, c2, c3 = (((p1 >> 32) & low) ^ c1 ^ k0, p1 & low,
                          ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), -1)


def _kept(s, c):
    n = c["rows"] * c["channels"]
    groups = torch.arange((n + 3) // 4, device="cuda")
    words = _philox(groups, s["seed"]).flatten()[:n]
    return (words >= int(c["p"] * 2 ** 32)).view(c["rows"], c["channels"])


def _plain_drop_forward(s, c):
    x = s["x"].float() * (1 / (1 - c["p"]))
    y = torch.where(_kept(s, c), x, torch.zeros_like(x))
    if s["residual"] is None:
        return {"y": y.to(s["x"].dtype)}
    return {"y": (s["residual"].float() + y).to(s["residual"].dtype)}


def _plain_drop_train(s, c):
    dy = s["dy"].float() * (1 / (1 - c["p"]))
    dx = torch.where(_kept(s, c), dy, torch.zeros_like(dy))
    return {**_plain_drop_forward(s, c), "dx": dx.to(s["x"].dtype)}


def _plain_ce(s, c):
    x, weight = s["x"].float(), s["weight"].float()
    logits = x @ weight.t()
    top = logits.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    counts = s["targets"] >= 0
    at = s["targets"].clamp(min=0)[:, None]
    zero = torch.zeros((), device="cuda")
    loss = torch.where(counts, (lse - logits.gather(1, at))[:, 0], zero)
    return x, weight, logits, lse, counts, at, zero, loss


def _plain_ce_forward(s, c):
    _, _, _, lse, counts, _, zero, loss = _plain_ce(s, c)
    return {"loss": loss, "lse": torch.where(counts, lse[:, 0], zero)}


def _plain_ce_train(s, c):
    x, weight, logits, lse, counts, at, zero, loss = _plain_ce(s, c)
    dloss = torch.where(counts, s["dloss"], zero)[:, None]
    both = dloss
    if s["dlse"] is not None:
        both = dloss + torch.where(counts, s["dlse"], zero)[:, None]
    grad = torch.exp(logits - lse) * both
    grad.scatter_add_(1, at, -dloss)
    return {"loss": loss, "lse": torch.where(counts, lse[:, 0], zero),
            "dx": (grad @ weight).to(s["x"].dtype),
            "dweight": (grad.t() @ x).to(s["weight"].dtype)}


_PLAIN = {("rec", "forward"): _plain_rec_forward, ("rec", "train"): _plain_rec_train,
          ("rec", "step"): _plain_rec_step, ("drop", "forward"): _plain_drop_forward,
          ("drop", "train"): _plain_drop_train, ("ce", "forward"): _plain_ce_forward,
          ("ce", "train"): _plain_ce_train}


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions in 64 bits: the recurrence as a product of its steps'
    maps by doubling, gradients by differentiation. Masks have no such value."""
    s = prepare(case, seed)
    wide = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v
            for k, v in s.items()}
    return _EXACT[case["op"]](wide, case)


def _leaf(v):
    return v.clone().requires_grad_(True)


def _exact_rec(s, c):
    train, step = c["mode"] == "train", c["mode"] == "step"
    x, ig, rg, decay, state = (s[k] for k in ("x", "ig", "rg", "decay", "state"))
    if step:
        x, ig, rg = x[:, None], ig[:, None], rg[:, None]
    if train:
        x, ig, rg, decay, state = map(_leaf, (x, ig, rg, decay, state))
    with torch.set_grad_enabled(train):
        log_a = -decay / (1 + torch.exp(-rg))
        keep = None if s["lengths"] is None else _inside(s, c)
        if keep is not None:
            log_a = log_a.masked_fill(~keep, 0.0)
        drive = torch.sqrt(-torch.expm1(2 * -decay / (1 + torch.exp(-rg)))) * x / (1 + torch.exp(-ig))
        if keep is not None:
            drive = drive.masked_fill(~keep, 0.0)
        # h[t] = f[t] h[t - span] + g[t], spans doubled until they reach the start
        f, g = torch.exp(log_a), drive
        g = torch.cat((g[:, :1] + f[:, :1] * state[:, None], g[:, 1:]), 1)
        span, n = 1, g.shape[1]
        while span < n:
            g = torch.cat((g[:, :span], g[:, span:] + f[:, span:] * g[:, :-span]), 1)
            f = torch.cat((f[:, :span], f[:, span:] * f[:, :-span]), 1)
            span *= 2
        out = g if keep is None else g.masked_fill(~keep, 0.0)
        if step:
            return {"out": out[:, 0], "state": g[:, 0]}
        res = {"out": out.detach(), "state": g[:, -1].detach()}
        if train:
            grads = torch.autograd.grad((out * s["dout"]).sum(), (x, ig, rg, decay, state))
            res.update(zip(("dx", "dig", "drg", "ddecay", "dstate"), grads))
    return res


def _exact_drop(s, c):
    factor = _kept(s, c).double() / (1 - c["p"])
    y = factor * s["x"]
    out = {"y": y if s["residual"] is None else s["residual"] + y}
    if c["mode"] == "train":
        out["dx"] = factor * s["dy"]
    return out


def _exact_ce(s, c):
    train = c["mode"] == "train"
    x, weight = (_leaf(s["x"]), _leaf(s["weight"])) if train else (s["x"], s["weight"])
    rows = torch.nonzero(s["targets"] >= 0)[:, 0]
    with torch.set_grad_enabled(train):
        logits = x[rows] @ weight.t()
        lse = torch.logsumexp(logits, 1)
        loss = lse - logits[torch.arange(len(rows), device="cuda"), s["targets"][rows]]
        whole = torch.zeros(c["tokens"], dtype=torch.float64, device="cuda")
        res = {"loss": whole.index_copy(0, rows, loss.detach()),
               "lse": whole.index_copy(0, rows, lse.detach())}
        if train:
            total = (loss * s["dloss"][rows]).sum()
            if s["dlse"] is not None:
                total = total + (lse * s["dlse"][rows]).sum()
            res["dx"], res["dweight"] = torch.autograd.grad(total, (x, weight))
    return res


_EXACT = {"rec": _exact_rec, "drop": _exact_drop, "ce": _exact_ce}


# ---------------------------------------------------------------- work

def work(case):
    e = _BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "rec":
        b, n, d = case["batch"], case["length"], case["channels"]
        if case.get("ragged"):       # about half of the steps lie inside
            n = (n + 1) // 2
        # three inputs and the output; with gradients the output's, and three
        size = b * n * d
        return {"bytes": size * e * (8 if train else 4) + b * d * (16 if train else 8) + d * 4,
                "flops": size * (45 if train else 18)}
    if case["op"] == "drop":
        size = case["rows"] * case["channels"]
        r = _BYTES[case["residual"]] if case["residual"] else 0
        y = r or e
        return {"bytes": size * ((e + r + y) + ((y + e) if train else 0)),
                "flops": size * (4 if train else 2)}
    t, d, v = case["tokens"], case["width"], case["vocab"]
    t_in = max(1, round(t * (1 - case["masked"])))
    return {"bytes": (t + v) * d * e * (2 if train else 1) + t * (20 if train else 16),
            "flops": t_in * d * v * (6 if train else 2)}
