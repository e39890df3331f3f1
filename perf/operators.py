"""The vocabulary's two ends of a language model, as cases that can be timed and checked.

  embedding   Y[n] = scale W[id[n]], and its gradient dW[v] = scale * sum of dY[n] over id[n] = v
  xent        softmax cross entropy of the logits H W^T against one target a row, with dH and dW
  distill     the same logits at a temperature against a teacher's K best logits a row, dH and dW

The table W (V x D) is the same thing in all three, and the gradients have its type.  An id or
target outside 0..V-1 is padding: a zero row, no loss and no gradient.  Each case is one pass
through an operator: forward and backward, or the forward alone where the case says so.

  own                   whether run() calls the framework's operators or their plain form
  listed()              the named cases
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   inputs, made from the seed, and the buffers that a program keeps
  run(state)            one pass; returns every output and gradient
  work(case)            bytes and floating-point operations that a pass cannot do without
  exact(case, seed)     the same outputs in 64 bits
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}
WORKSPACE = 2 << 30   # what a training program sets aside for its largest operator


def listed():
    return [
        # A character-level model: the smallest table and batch, where launches are what counts.
        dict(name="embed_char_f32", op="embedding", dtype="f32", N=256, V=65, D=32, pad=0.0,
             grad=True),
        # A training batch over an ordinary table; padded sequences, odd number of rows in it.
        dict(name="embed_train_bf16", op="embedding", dtype="bf16", N=8192, V=50001, D=1024,
             pad=0.06, grad=True),
        # A long batch over a wide table in the default precision: the largest.
        dict(name="embed_large_f32", op="embedding", dtype="f32", N=65536, V=131072, D=2048,
             pad=0.0, grad=True),
        # The loss of that character-level model.
        dict(name="xent_char_f32", op="xent", dtype="f32", N=256, V=65, D=32, pad=0.0, grad=True),
        # A training step in the default precision.
        dict(name="xent_train_f32", op="xent", dtype="f32", N=2048, V=32000, D=1024, pad=0.0,
             grad=True),
        # A training step over padded sequences, odd table and width that end inside a tile.
        dict(name="xent_ragged_bf16", op="xent", dtype="bf16", N=4001, V=50001, D=1000, pad=0.1,
             grad=True),
        # A training step over a large vocabulary: the largest.
        dict(name="xent_large_bf16", op="xent", dtype="bf16", N=8192, V=131072, D=2048, pad=0.0,
             grad=True),
        # Scoring of a text without gradients.
        dict(name="xent_score_bf16", op="xent", dtype="bf16", N=1024, V=131072, D=4096, pad=0.0,
             grad=False),
        # The log-probability of a single token: the table is read once, little is computed.
        dict(name="xent_token_bf16", op="xent", dtype="bf16", N=1, V=131072, D=2048, pad=0.0,
             grad=False),
        # A small student in the default precision, few teacher logits.
        dict(name="distill_small_f32", op="distill", dtype="f32", N=200, V=1000, D=128, K=8,
             pad=0.0, T=2.0, grad=True),
        # A student's training step.
        dict(name="distill_train_bf16", op="distill", dtype="bf16", N=2048, V=32000, D=1024, K=32,
             pad=0.05, T=2.0, grad=True),
        # The same over a large vocabulary with many teacher logits.
        dict(name="distill_large_bf16", op="distill", dtype="bf16", N=4096, V=131072, D=2048,
             K=100, pad=0.0, T=1.0, grad=True),
    ]


# --------------------------------------------------------------------------- drawing

def _size(rng, lo, hi):
    """A size of lo..hi, even over its logarithm: half of them a multiple of 16 (where that
    fits), half as they come."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v = v // 16 * 16
    return max(lo, min(hi, v))


def _seconds(case):
    """A rough estimate of a pass of the plain form."""
    w = work(case)
    return w["flops"] / 100e12 + w["bytes"] / 1e12


def _draw(rng):
    op = rng.choice(("embedding", "xent", "xent", "distill"))
    c = dict(op=op, dtype=rng.choice(("f32", "bf16")))
    if op == "embedding":
        c.update(N=_size(rng, 1, 65536), V=_size(rng, 2, 131072), D=_size(rng, 16, 4096))
    else:
        c.update(N=_size(rng, 1, 16384), V=_size(rng, 16, 131072), D=_size(rng, 16, 4096))
    if op == "distill":
        c.update(K=_size(rng, 1, min(128, c["V"])), T=rng.choice((1.0, 2.0, 4.0)))
    c.update(pad=rng.choice((0.0, 0.0, round(rng.uniform(0.02, 0.5), 2))),
             grad=op != "xent" or rng.random() < 0.7)
    return c


def draw(rng):
    most = max(_seconds(c) for c in listed())
    while True:
        c = _draw(rng)
        if _seconds(c) <= most:
            return c


# --------------------------------------------------------------------------- inputs

def _ids(g, N, V, pad):
    """Tokens as text has them: frequent ones first, rank r about as often as 1 / r; a share
    `pad` of them, at the end, is padding (-1)."""
    u = torch.rand(N, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(V)).floor() - 1).clamp_(0, V - 1).to(torch.int32)
    if pad:
        ids[N - int(round(N * pad)):] = -1
    return ids


def _inputs(c, seed):
    """The tensors that a pass reads, by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, V, D, dt = c["N"], c["V"], c["D"], TORCH[c["dtype"]]
    W = torch.randn((V, D), generator=g, device="cuda").mul_(0.02)
    t = dict(W=W.to(dt), ids=_ids(g, N, V, c["pad"]))
    del W
    if c["op"] == "embedding":
        t["dY"] = torch.randn((N, D), generator=g, device="cuda").mul_(1e-3).to(dt)
        return t
    # Normed hidden states that lean towards their target: logits of a spread of 2 to 3, the
    # target's probability anywhere between 0 and 1.
    H = torch.randn((N, D), generator=g, device="cuda") * (2.5 / (0.02 * math.sqrt(D)))
    lean = t["W"][t["ids"].clamp(min=0).long()].float()
    H += lean * (torch.rand((N, 1), generator=g, device="cuda") * 12.0
                 / (0.0004 * D))
    t["H"] = H.to(dt)
    # Each row counts for its share of the mean, as a training loss weighs it.
    t["dloss"] = torch.full((N,), 1.0 / N, device="cuda")
    if c["op"] == "distill":
        K = c["K"]
        # K different tokens a row, the target the first of them, and logits that fall off.
        first = t["ids"].clamp(min=0).long()[:, None]
        idx = (first + torch.arange(K, device="cuda")[None, :] * (V // K)) % V
        top = torch.randn((N, K), generator=g, device="cuda") * 2.0 + 10.0
        t["top_logit"] = top.sort(dim=1, descending=True).values
        t["top_id"] = torch.where(t["ids"][:, None] < 0, -1, idx).to(torch.int32)
    return t


class State:
    """A case's inputs, output buffers and workspace."""

    def __init__(self, case, seed):
        self.case = case
        self.t = t = _inputs(case, seed)
        N, D, dt = case["N"], case["D"], TORCH[case["dtype"]]
        if case["op"] == "embedding":
            t["Y"] = torch.empty((N, D), dtype=dt, device="cuda")
        else:
            t["loss"] = torch.empty(N, device="cuda")
            t["lse"] = torch.empty(N, device="cuda")
            if case["grad"]:
                t["dH"] = torch.empty((N, D), dtype=dt, device="cuda")
        if case["grad"]:
            t["dW"] = torch.empty_like(t["W"])
        t["ws"] = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
        self.p = {n: x.data_ptr() for n, x in t.items()}
        torch.cuda.synchronize()   # the library has a stream of its own


def prepare(case, seed):
    return State(case, seed)


# --------------------------------------------------------------------------- one pass

def _scale(c):
    """The embedding's factor, sqrt(D), as models with a shared table use it."""
    return math.sqrt(c["D"])


def _run_own(s):
    from dreamcompiler_amd import hip
    c, t, p = s.case, s.t, s.p
    N, V, D = c["N"], c["V"], c["D"]
    dt = hip.F32 if c["dtype"] == "f32" else hip.BF16
    if c["op"] == "embedding":
        hip.embedding_fwd(dt, N, V, D, _scale(c), p["ids"], p["W"], D, p["Y"], D)
        hip.embedding_bwd(dt, N, V, D, _scale(c), p["ids"], p["dY"], D, p["dW"], D, dt, False,
                          p["ws"], WORKSPACE)
        return [t["Y"], t["dW"]]
    if c["op"] == "xent":
        a = (dt, N, V, D, 1.0, p["H"], D, p["W"], D, p["ids"])
        hip.linear_xent_fwd(*a, p["loss"], p["lse"], p["ws"], WORKSPACE)
        if not c["grad"]:
            return [t["loss"], t["lse"]]
        hip.linear_xent_bwd(*a, p["lse"], p["dloss"], p["dH"], D, False, p["dW"], D, False, dt,
                            p["ws"], WORKSPACE)
    else:
        a = (dt, N, V, D, c["K"], c["T"], p["H"], D, p["W"], D, p["top_id"], p["top_logit"])
        hip.linear_distill_fwd(*a, p["loss"], p["lse"], p["ws"], WORKSPACE)
        hip.linear_distill_bwd(*a, p["lse"], p["dloss"], p["dH"], D, False, p["dW"], D, False, dt,
                               p["ws"], WORKSPACE)
    return [t[n] for n in ("loss", "lse", "dH", "dW")]


def _run_plain(s):
    c, t = s.case, s.t
    V, dt = c["V"], TORCH[c["dtype"]]
    if c["op"] == "embedding":
        valid = (t["ids"] >= 0)[:, None]
        ids = t["ids"].clamp(min=0).long()
        Y = torch.where(valid, t["W"][ids].float() * _scale(c), 0.0).to(dt)
        dY = torch.where(valid, t["dY"].float() * _scale(c), 0.0)
        dW = torch.zeros((V, c["D"]), device="cuda").index_add_(0, ids, dY)
        return [Y, dW.to(dt)]
    H, W = t["H"].float(), t["W"].float()
    scale = 1.0 if c["op"] == "xent" else 1.0 / c["T"]
    z = (H @ W.t()) * scale
    m = z.max(dim=1, keepdim=True).values
    e = (z - m).exp()
    total = e.sum(dim=1, keepdim=True)
    lse = m + total.log()
    if c["op"] == "xent":
        valid = (t["ids"] >= 0)[:, None]
        at = t["ids"].clamp(min=0).long()[:, None]
        q = torch.ones_like(at, dtype=torch.float32)
        loss = lse - z.gather(1, at)
    else:
        valid = t["top_id"][:, :1] >= 0
        at = t["top_id"].clamp(min=0).long()
        y = t["top_logit"] * scale
        q = (y - y.max(dim=1, keepdim=True).values).exp()
        q = q / q.sum(dim=1, keepdim=True)
        loss = (q * (q.log() - z.gather(1, at) + lse)).sum(dim=1, keepdim=True) / scale ** 2
    out = [torch.where(valid, loss, 0.0)[:, 0], torch.where(valid, lse, 0.0)[:, 0]]
    if not c["grad"]:
        return out
    del z
    w = torch.where(valid, t["dloss"][:, None] / (1.0 if c["op"] == "xent" else scale), 0.0)
    G = e.mul_(w / total).scatter_add_(1, at, -w * q)
    return out + [(G @ W).to(dt), (G.t() @ H).to(dt)]


def run(s):
    return _run_own(s) if own else _run_plain(s)


# --------------------------------------------------------------------------- what a pass needs

def work(c):
    N, V, D, e = c["N"], c["V"], c["D"], BYTES[c["dtype"]]
    if c["op"] == "embedding":
        # ids, at most N rows of the table, Y and dY, the whole gradient
        return {"bytes": 4 * N + e * D * (min(N, V) + 2 * N + V), "flops": 2 * N * D}
    rows = N - int(round(N * c["pad"]))   # padding has no product
    n = N * D + V * D
    return {"bytes": e * n * (2 if c["grad"] else 1) + 16 * N + 8 * N * c.get("K", 0),
            "flops": (6 if c["grad"] else 2) * rows * V * D}


# --------------------------------------------------------------------------- in 64 bits

def exact(c, seed):
    t = _inputs(c, seed)
    V, D = c["V"], c["D"]
    if c["op"] == "embedding":
        keep = t["ids"] >= 0
        ids = t["ids"][keep].long()
        Y = torch.zeros((c["N"], D), dtype=torch.float64, device="cuda")
        Y[keep] = t["W"].double()[ids] * _scale(c)
        # Tokens in the order of their ids, and the sum of each run.
        order = torch.argsort(ids, stable=True)
        rows, count = torch.unique_consecutive(ids[order], return_counts=True)
        dW = torch.zeros((V, D), dtype=torch.float64, device="cuda")
        if rows.numel():
            dW[rows] = torch.segment_reduce(t["dY"][keep][order].double(), "sum",
                                            lengths=count) * _scale(c)
        return [Y, dW]
    W = t["W"].double()
    loss = torch.zeros(c["N"], dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(loss)
    dH = torch.zeros((c["N"], D), dtype=torch.float64, device="cuda")
    dW = torch.zeros_like(W)
    keep = torch.nonzero(t["ids"] >= 0)[:, 0]
    temp = c.get("T", 1.0)
    for rows in keep.split(2048):
        Hr = t["H"][rows].double()
        logp = torch.log_softmax(Hr @ W.t() / temp, dim=1)
        lse[rows] = (Hr[:, None, :] * W[t["ids"][rows].long()][:, None, :]).sum(-1)[:, 0] / temp \
            - logp.gather(1, t["ids"][rows].long()[:, None])[:, 0]
        target = torch.zeros_like(logp)
        if c["op"] == "xent":
            target[torch.arange(len(rows), device="cuda"), t["ids"][rows].long()] = 1.0
            loss[rows] = -(target * logp).sum(1)
        else:
            logq = torch.log_softmax(t["top_logit"][rows].double() / temp, dim=1)
            at = t["top_id"][rows].long()
            target.scatter_(1, at, logq.exp())
            loss[rows] = temp ** 2 * (logq.exp() * (logq - logp.gather(1, at))).sum(1)
        if c["grad"]:
            G = logp.exp_().sub_(target).mul_(t["dloss"][rows].double()[:, None] * temp)
            dH[rows] = G @ W
            dW += G.t() @ Hr
    return [loss, lse, dH, dW] if c["grad"] else [loss, lse]
