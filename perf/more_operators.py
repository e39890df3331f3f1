"""What a decoder's attention needs around the flash kernels, as cases that can be timed and checked.

  qk       RMS norm of every head's query and key, times a weight, and the rotation by position,
           from the projections' rows into attention's layout; with its gradient
  cache    keys and values of new tokens into a paged cache (rounded to 8 bits with a scale for
           each token and head where the cache's type has them), and read back for attention over
           whole sequences
  decode   attention of one new token of each sequence over such a cache

A cache holds pages x Hk x page x D values (keys and values apart) and, for 8-bit types, as many
scales without the D; sequence b's token t is in page table[b, t // page].  Each case is one pass
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

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8,
         "f8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "i8": 1, "f8": 1}
TOP = {"i8": 127.0, "f8": 448.0}    # a row's largest value, over its scale
EPS = 1e-6
BASE = 10000.0
WORKSPACE = 256 << 20   # what a program sets aside for these operators


def listed():
    return [
        # The token that a single sequence goes on with: launches are what counts.
        dict(name="qk_token_bf16", op="qk", dtype="bf16", B=1, S=1, Hq=32, Hk=8, D=128, R=128,
             pairs=False, pad=0.0, grad=False),
        # A prompt of many tokens with fewer heads of keys than of queries.
        dict(name="qk_prompt_bf16", op="qk", dtype="bf16", B=1, S=16384, Hq=32, Hk=8, D=128,
             R=128, pairs=False, pad=0.0, grad=False),
        # A training step in fp32 over a padded batch: odd sizes, neighbours as pairs, a part of
        # each head turned.
        dict(name="qk_ragged_f32", op="qk", dtype="f32", B=3, S=1333, Hq=12, Hk=3, D=80, R=40,
             pairs=True, pad=0.1, grad=True),
        # The training step of the benchmark's attention shape.
        dict(name="qk_train_bf16", op="qk", dtype="bf16", B=8, S=4096, Hq=16, Hk=16, D=128,
             R=128, pairs=False, pad=0.0, grad=True),
        # One token of each sequence of a batch goes into an 8-bit cache.
        dict(name="cache_token_i8", op="cache", dtype="bf16", cache="i8", B=64, longest=4096,
             new=1, read=1, Hk=8, D=128, page=16),
        # Odd prompts in fp32, kept in 8-bit integers, read back whole.
        dict(name="cache_ragged_i8", op="cache", dtype="f32", cache="i8", B=5, longest=1999,
             new=777, read=1999, Hk=3, D=80, page=32),
        # A piece of long prompts, kept in 8-bit floats; attention over all of them reads back.
        dict(name="cache_prompt_f8", op="cache", dtype="bf16", cache="f8", B=8, longest=16384,
             new=4096, read=16384, Hk=8, D=128, page=64),
        # A single short sequence, a head of keys for each of queries.
        dict(name="decode_short_bf16", op="decode", dtype="bf16", cache="bf16", B=1, longest=512,
             Hq=16, Hk=16, D=128, page=16, window=0, empty=False),
        # A single long sequence: split over its length, or most of the GPU idles.
        dict(name="decode_long_bf16", op="decode", dtype="bf16", cache="bf16", B=1,
             longest=131072, Hq=32, Hk=8, D=128, page=16, window=0, empty=False),
        # A padded fp32 batch with odd lengths that sees the last 1000 tokens.
        dict(name="decode_ragged_f32", op="decode", dtype="f32", cache="f32", B=33, longest=2047,
             Hq=12, Hk=12, D=64, page=32, window=1000, empty=True),
        # A serving batch of sequences of many lengths, in the model's type and in 8 bits.
        dict(name="decode_batch_bf16", op="decode", dtype="bf16", cache="bf16", B=64,
             longest=8192, Hq=32, Hk=8, D=128, page=16, window=0, empty=False),
        dict(name="decode_batch_f8", op="decode", dtype="bf16", cache="f8", B=128, longest=8192,
             Hq=64, Hk=8, D=128, page=64, window=0, empty=False),
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
    op = rng.choice(("qk", "cache", "decode", "decode"))
    dtype = rng.choice(("f32", "bf16"))
    Hk = rng.choice((1, 2, 3, 4, 8, 16))
    if op == "qk":
        D = rng.choice((32, 64, 80, 96, 100, 128, 192, 256))
        return dict(op=op, dtype=dtype, B=_size(rng, 1, 16), S=_size(rng, 1, 16384),
                    Hq=Hk * rng.choice((1, 1, 2, 4, 8)), Hk=Hk, D=D,
                    R=rng.choice((D, D, D // 4 * 2)), pairs=rng.random() < 0.5,
                    pad=rng.choice((0.0, 0.0, round(rng.uniform(0.02, 0.5), 2))),
                    grad=rng.random() < 0.6)
    c = dict(op=op, dtype=dtype, cache=rng.choice((dtype, "i8", "f8")), B=_size(rng, 1, 128),
             longest=_size(rng, 1, 131072))
    if op == "decode":
        c["Hq"] = Hk * rng.choice((1, 2, 4, 5, 8, 16, 20))
    c.update(Hk=Hk, D=rng.choice((32, 64, 80, 96, 128, 128, 192, 256)),
             page=rng.choice((16, 32, 64, 128, 256)))
    if op == "decode":
        c.update(window=rng.choice((0, 0, _size(rng, 1, c["longest"]))),
                 empty=rng.random() < 0.3)
    else:
        c["new"] = rng.choice((1, _size(rng, 1, c["longest"])))
        c["read"] = rng.choice((c["new"], c["longest"]))
    return c


def draw(rng):
    most = max(_seconds(c) for c in listed())
    while True:
        c = _draw(rng)
        if _seconds(c) <= most:
            return c


# --------------------------------------------------------------------------- inputs

def _lengths(c):
    """The sequences' lengths, from the longest down to an eighth of it, evenly; the last one is
    empty where the case says so."""
    B, top = c["B"], c["longest"]
    lens = [max(1, round(top * (1.0 - 0.875 * b / B))) for b in range(B)]
    if c.get("empty") and B > 1:
        lens[-1] = 0
    return lens


def _rows(lens, most):
    """For each sequence its last tokens, `most` of them at most."""
    return [min(n, most) for n in lens]


def _first(counts):
    """Where each sequence's rows begin, and their end."""
    t = torch.zeros(len(counts) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
    return t.cuda()


def _rope_table(P, R):
    """Cosines and sines of p * BASE^(-2 i / R), P x R, side by side."""
    i = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * BASE ** (-2.0 * i / R)
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _fill_cache(t, c, g):
    """Pages that hold what such a cache holds: values in the type itself, or 8-bit ones up to the
    type's largest and scales of their rows."""
    shape = (t["pages"], c["Hk"], c["page"], c["D"])
    for n in ("Kc", "Vc"):
        if c["cache"] in TOP:
            top = TOP[c["cache"]]
            x = torch.randn(shape, generator=g, device="cuda").mul_(top / 4.0)
            x = x.round_() if c["cache"] == "i8" else x
            t[n] = x.clamp_(-top, top).to(TORCH[c["cache"]]).view(torch.uint8)
            s = torch.rand(shape[:3], generator=g, device="cuda") + 0.5
            t[n[0] + "s"] = s * (4.0 / top)
        else:
            t[n] = torch.empty(shape, dtype=TORCH[c["cache"]], device="cuda").normal_(generator=g)
            t[n[0] + "s"] = None


def _inputs(c, seed):
    """The tensors that a pass reads, by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, D = TORCH[c["dtype"]], c["D"]
    if c["op"] == "qk":
        B, S, R, heads = c["B"], c["S"], c["R"], c["Hq"] + 2 * c["Hk"]
        # The projections' output: a token's queries, keys and values side by side.
        t = dict(X=torch.empty((B, S, heads, D), dtype=dt, device="cuda").normal_(generator=g))
        t["gq"], t["gk"] = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")
                            for _ in range(2))
        t["pos"] = torch.arange(S, device="cuda", dtype=torch.int32).repeat(B, 1)
        # What lies behind a sequence's end is padding.
        if c["pad"]:
            t["pos"][:, S - int(round(S * c["pad"])):] = -1
        t["P"] = S
        t["table"] = _rope_table(S, R)
        if c["grad"]:
            for n, H in (("dQo", c["Hq"]), ("dKo", c["Hk"])):
                # What the flash backward leaves: fp32, in its own layout.
                t[n] = torch.randn((B, H, S, D), generator=g, device="cuda") * 1e-2
        return t
    t = {}
    lens = _lengths(c)
    order = torch.randperm(c["B"], generator=g, device="cuda").tolist()
    lens = [lens[i] for i in order]
    t["len_list"] = lens
    t["len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    held = [-(-n // c["page"]) for n in lens]
    t["pages"] = sum(held) + 7      # some are free
    t["ld"] = max(1, max(held))
    t["table"] = torch.full((c["B"], t["ld"]), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(t["pages"], generator=g, device="cuda").to(torch.int32)
    slot = torch.arange(t["ld"], device="cuda")[None, :] < torch.tensor(held).cuda()[:, None]
    t["table"][slot] = ids[:sum(held)]
    _fill_cache(t, c, g)
    if c["op"] == "cache":
        new, read = _rows(lens, c["new"]), _rows(lens, c["read"])
        t["N"], t["M"] = sum(new), sum(read)
        t["new"], t["read"] = _first(new), _first(read)
        # Keys and values of the projections' output, beside each other; some heads are louder.
        t["KV"] = torch.randn((t["N"], 2, c["Hk"], D), generator=g, device="cuda")
        t["KV"] *= torch.exp2(torch.randint(-3, 4, (t["N"], 2, c["Hk"], 1), generator=g,
                                            device="cuda").float())
        t["KV"] = t["KV"].to(dt)
    else:
        # Heads that look at everything alike, and heads that look at a few tokens.
        sharp = torch.rand((1, c["Hq"], 1), generator=g, device="cuda") * 3.5 + 0.5
        t["Q"] = (torch.randn((c["B"], c["Hq"], D), generator=g, device="cuda") * sharp).to(dt)
    return t


class State:
    """A case's inputs, output buffers and workspace."""

    def __init__(self, case, seed):
        self.case = case
        self.t = t = _inputs(case, seed)
        dt, D = TORCH[case["dtype"]], case["D"]
        new = lambda shape, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
        if case["op"] == "qk":
            B, S = case["B"], case["S"]
            t["Qo"], t["Ko"] = new((B, case["Hq"], S, D)), new((B, case["Hk"], S, D))
            if case["grad"]:
                t["dX"] = torch.zeros_like(t["X"])
                t["dgq"], t["dgk"] = new(D, torch.float32), new(D, torch.float32)
        elif case["op"] == "cache":
            t["K"], t["V"] = (new((t["M"], case["Hk"], D)) for _ in range(2))
        else:
            t["O"] = torch.empty_like(t["Q"])
            t["lse"] = new((case["B"], case["Hq"]), torch.float32)
        t["ws"] = new(WORKSPACE, torch.uint8)
        self.p = {n: x.data_ptr() for n, x in t.items() if isinstance(x, torch.Tensor)}
        torch.cuda.synchronize()   # the library has a stream of its own


def prepare(case, seed):
    return State(case, seed)


# --------------------------------------------------------------------------- one pass

def _scale(c):
    return 1.0 / math.sqrt(c["D"])


def _run_own(s):
    from dreamcompiler_amd import hip
    c, t, p = s.case, s.t, s.p
    D, Hk = c["D"], c["Hk"]
    types = {"f32": hip.F32, "bf16": hip.BF16, "i8": hip.I8, "f8": hip.F8}
    dt, e = types[c["dtype"]], BYTES[c["dtype"]]
    if c["op"] == "qk":
        B, S, Hq = c["B"], c["S"], c["Hq"]
        row = (Hq + 2 * Hk) * D
        wide = (S * row, row, D)                   # sequence, token, head
        of_q, of_k = (Hq * S * D, D, S * D), (Hk * S * D, D, S * D)
        a = (dt, B, S, Hq, Hk, D, c["R"], c["pairs"], EPS, p["pos"], p["table"], t["P"],
             p["X"], wide, p["X"] + Hq * D * e, wide, p["gq"], p["gk"])
        hip.qk_norm_rope_fwd(*a, p["Qo"], of_q, p["Ko"], of_k)
        if not c["grad"]:
            return [t["Qo"], t["Ko"]]
        hip.qk_norm_rope_bwd(*a, hip.F32, p["dQo"], of_q, p["dKo"], of_k, dt, p["dX"], wide,
                             p["dX"] + Hq * D * e, wide, p["dgq"], p["dgk"], False, p["ws"],
                             WORKSPACE)
        return [t["Qo"], t["Ko"], t["dX"][:, :, :Hq], t["dX"][:, :, Hq:Hq + Hk], t["dgq"],
                t["dgk"]]
    held = (t["pages"], c["page"], p["table"], t["ld"], p["Kc"], p["Vc"], p.get("Ks"),
            p.get("Vs"))
    if c["op"] == "cache":
        kv, out = (2 * Hk * D, D), (Hk * D, D)     # token, head
        hip.kv_cache_write(dt, types[c["cache"]], c["B"], t["N"], Hk, D, p["KV"], kv,
                           p["KV"] + Hk * D * e, kv, p["new"], p["len"], *held)
        hip.kv_cache_read(dt, types[c["cache"]], c["B"], t["M"], Hk, D, p["K"], out, p["V"], out,
                          p["read"], p["len"], *held)
        return [t["K"], t["V"]]
    one = (c["Hq"] * D, D)                         # sequence, head
    hip.paged_attention(dt, types[c["cache"]], c["B"], c["Hq"], Hk, D, _scale(c), c["window"],
                        p["Q"], one, p["len"], c["longest"], *held, p["O"], one, p["lse"],
                        p["ws"], WORKSPACE)
    return [t["O"], t["lse"]]


def _turn(c, y, cos, sin):
    """y (B x S x H x D) with its first R values turned."""
    R = c["R"]
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if c["pairs"] else (y[..., :R // 2], y[..., R // 2:R])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], dim=-1).flatten(-2) if c["pairs"] else torch.cat([u, v], dim=-1)
    return torch.cat([turned, y[..., R:]], dim=-1)


def _plain_qk(c, t):
    S, R, Hq, Hk, dt = c["S"], c["R"], c["Hq"], c["Hk"], TORCH[c["dtype"]]
    there = (t["pos"] >= 0)[:, :, None, None]
    angle = t["table"][t["pos"].clamp(min=0).long()][:, :, None, :]
    cos, sin = angle[..., :R // 2], angle[..., R // 2:]

    def forward(x, w):
        r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
        out = _turn(c, x * r * w, cos, sin)
        return r, torch.where(there, out, 0.0).transpose(1, 2).to(dt).contiguous()

    def backward(x, w, r, dout):
        dy = _turn(c, torch.where(there, dout.transpose(1, 2), 0.0), cos, -sin)
        xr = x * r
        dw = (dy * xr).sum(dim=(0, 1, 2))
        dy = dy * w
        return ((dy - xr * (dy * xr).mean(dim=-1, keepdim=True)) * r).to(dt), dw

    q, k = t["X"][:, :, :Hq].float(), t["X"][:, :, Hq:Hq + Hk].float()
    rq, Qo = forward(q, t["gq"])
    rk, Ko = forward(k, t["gk"])
    if not c["grad"]:
        return [Qo, Ko]
    dQ, dgq = backward(q, t["gq"], rq, t["dQo"])
    dK, dgk = backward(k, t["gk"], rk, t["dKo"])
    return [Qo, Ko, dQ, dK, dgq, dgk]


def _places(c, t, first, n):
    """Page and place in it of rows 0..n-1, of which sequence b has first[b]..first[b+1]-1: its last
    tokens."""
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(first[1:].contiguous(), row, right=True)
    at = (t["len"][b] - (first[b + 1] - row)).long()
    return t["table"][b, at // c["page"]].long(), at % c["page"]


def _round_f8(y):
    """y (64 bits) to the nearest e4m3 value, ties to the even one."""
    step = torch.exp2((torch.frexp(y)[1] - 4).clamp(min=-9).double())
    return (torch.round(y / step) * step).float()


def _plain_cache(c, t):
    D, Hk, kind, dt = c["D"], c["Hk"], c["cache"], TORCH[c["dtype"]]
    page, at = _places(c, t, t["new"], t["N"])
    heads = torch.arange(Hk, device="cuda")[None, :]
    to = (page[:, None], heads, at[:, None])
    K, V = t["KV"][:, 0], t["KV"][:, 1]

    def write(x, pages, scales):
        if kind in TOP:
            # In 64 bits: quotients lie next to the borders between two 8-bit values.
            s = (x.double().abs().amax(dim=-1) / TOP[kind]).float()
            y = x.double() / torch.where(s > 0, s, 1.0).double()[..., None]
            x = torch.round(y) if kind == "i8" else _round_f8(y)
            x = x.clamp(-TOP[kind], TOP[kind]).to(TORCH[kind]).view(torch.uint8)
            scales[to] = s
        pages[to] = x

    def read(pages, scales):
        x = pages[src]
        if kind in TOP:
            x = x.view(TORCH[kind]).float() * scales[src][..., None]
        return x.to(dt)

    write(K, t["Kc"], t["Ks"])
    write(V, t["Vc"], t["Vs"])
    page, at = _places(c, t, t["read"], t["M"])
    src = (page[:, None], heads, at[:, None])
    return [read(t["Kc"], t["Ks"]), read(t["Vc"], t["Vs"])]


def _plain_decode(c, t):
    B, Hq, Hk, D, L = c["B"], c["Hq"], c["Hk"], c["D"], t["ld"] * c["page"]
    pages = t["table"].clamp(min=0).long()
    at = torch.arange(L, device="cuda")[None, :]
    seen = at < t["len"][:, None]
    if c["window"]:
        seen = seen & (at >= t["len"][:, None] - c["window"])

    def held(x, scales):
        y = x[pages]                                             # B x ld x Hk x page x D
        if c["cache"] in TOP:
            y = y.view(TORCH[c["cache"]]).float() * scales[pages][..., None]
        return y.float().transpose(1, 2).reshape(B * Hk, L, D)

    q = t["Q"].float().reshape(B * Hk, Hq // Hk, D) * _scale(c)
    z = torch.bmm(q, held(t["Kc"], t["Ks"]).transpose(1, 2).contiguous()).reshape(B, Hq, L)
    z = torch.where(seen[:, None, :], z, -math.inf)
    m = z.amax(dim=-1, keepdim=True)
    e = torch.where(seen[:, None, :], (z - m).exp(), 0.0)
    total = e.sum(dim=-1, keepdim=True)
    lse = torch.where(total > 0, m + total.log(), -math.inf)[..., 0]
    p = (e / torch.where(total > 0, total, 1.0)).reshape(B * Hk, Hq // Hk, L)
    O = torch.bmm(p, held(t["Vc"], t["Vs"])).reshape(B, Hq, D)
    O = torch.where((t["len"] > 0)[:, None, None], O, 0.0)
    return [O.to(TORCH[c["dtype"]]), lse]


def run(s):
    if own:
        return _run_own(s)
    return {"qk": _plain_qk, "cache": _plain_cache, "decode": _plain_decode}[s.case["op"]](
        s.case, s.t)


# --------------------------------------------------------------------------- what a pass needs

def work(c):
    D, e = c["D"], BYTES[c["dtype"]]
    if c["op"] == "qk":
        rows, values = c["B"] * c["S"], c["B"] * c["S"] * (c["Hq"] + c["Hk"]) * D
        n = 2 * e * values + 4 * (rows + c["S"] * c["R"] + 2 * D)
        if c["grad"]:   # inputs and the rotation's table again, fp32 gradients in, gradients out
            n += (2 * e + 4) * values + 4 * (rows + c["S"] * c["R"] + 4 * D)
        return {"bytes": n, "flops": values * (26 if c["grad"] else 9)}
    lens, f, scaled = _lengths(c), BYTES[c["cache"]], 4 if c["cache"] in TOP else 0
    if c["op"] == "cache":
        row = 2 * c["Hk"] * (D * (e + f) + scaled)
        n = sum(_rows(lens, c["new"])) + sum(_rows(lens, c["read"]))
        return {"bytes": n * row, "flops": n * 4 * c["Hk"] * D}
    seen = sum(min(n, c["window"]) if c["window"] else n for n in lens)
    return {"bytes": seen * 2 * c["Hk"] * (D * f + scaled) + c["B"] * c["Hq"] * (2 * D * e + 4),
            "flops": seen * 4 * c["Hq"] * D}


# --------------------------------------------------------------------------- in 64 bits

def _exact_qk(c, t):
    R, S, Hq, Hk = c["R"], c["S"], c["Hq"], c["Hk"]
    i = torch.arange(R // 2, device="cuda")
    at, with_ = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + R // 2)
    rows = t["table"].double()
    pos = t["pos"].flatten()
    there = (pos >= 0).nonzero()[:, 0]
    angle = torch.complex(rows[:, :R // 2], rows[:, R // 2:])[pos[there].long()][:, None, :]
    out, grads = [], []
    for lo, H, w, dname in ((0, Hq, t["gq"], "dQo"), (Hq, Hk, t["gk"], "dKo")):
        x = t["X"].flatten(0, 1)[there, lo:lo + H].double()
        norm = (x.square().sum(-1, keepdim=True) / c["D"] + EPS).sqrt()
        y = x / norm * w.double()
        z = torch.complex(y[..., at], y[..., with_]) * angle
        y[..., at], y[..., with_] = z.real, z.imag
        full = torch.zeros((len(pos), H, c["D"]), dtype=torch.float64, device="cuda")
        full[there] = y
        out.append(full.unflatten(0, (c["B"], S)).transpose(1, 2))
        if not c["grad"]:
            continue
        d = t[dname].transpose(1, 2).flatten(0, 1)[there].double()
        z = torch.complex(d[..., at], d[..., with_]) * angle.conj()
        d[..., at], d[..., with_] = z.real, z.imag
        dw = (d * x / norm).sum((0, 1))
        d *= w.double()
        # d(x / norm): the part along x goes
        along = (d * x).sum(-1, keepdim=True) / (c["D"] * norm.square())
        full = torch.zeros_like(full)
        full[there] = (d - along * x) / norm
        grads.append((full.unflatten(0, (c["B"], S)), dw))
    if not c["grad"]:
        return out
    return out + [grads[0][0], grads[1][0], grads[0][1], grads[1][1]]


def _codes_f8():
    """The e4m3 values from 0 up, in the order of their codes."""
    code = torch.arange(127, device="cuda", dtype=torch.uint8)
    return code.view(torch.float8_e4m3fn).double()


def _exact_rounded(c, x):
    """x's 8-bit values times their scales, from the definition."""
    x = x.double()
    s = (x.abs().amax(-1, keepdim=True) / TOP[c["cache"]]).float().double()
    if c["cache"] == "i8":
        values = torch.arange(128, device="cuda", dtype=torch.float64)
    else:
        values = _codes_f8()
    between = (values[1:] + values[:-1]) / 2
    y = torch.where(s > 0, x.abs() / s, 0.0)
    n = torch.searchsorted(between, y)
    tie = (n < len(between)) & (y == between[n.clamp(max=len(between) - 1)]) & (n % 2 == 1)
    return torch.sign(x) * values[n + tie] * s


def _exact_cache(c, t):
    out = []
    sides = ((0, t["Kc"], t["Ks"]), (1, t["Vc"], t["Vs"]))
    new, read = t["new"].tolist(), t["read"].tolist()
    for side, pages, scales in sides:
        rows = []
        for b, n in enumerate(t["len_list"]):
            ids = t["table"][b, :-(-n // c["page"])].long()
            x = pages[ids]
            if c["cache"] in TOP:
                x = x.view(TORCH[c["cache"]]).double() * scales[ids].double()[..., None]
            x = x.double().transpose(1, 2).reshape(-1, c["Hk"], c["D"])[:n]
            fresh = t["KV"][new[b]:new[b + 1], side]
            if c["cache"] in TOP:
                fresh = _exact_rounded(c, fresh)
            x[n - (new[b + 1] - new[b]):] = fresh.double()
            rows.append(x[n - (read[b + 1] - read[b]):])
        out.append(torch.cat(rows))
    return out


def _exact_decode(c, t):
    O = torch.zeros(t["Q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(t["Q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(t["len_list"]):
        if n == 0:
            continue
        ids = t["table"][b, :-(-n // c["page"])].long()
        since = max(0, n - c["window"]) if c["window"] else 0
        K, V = (pages[ids] for pages in (t["Kc"], t["Vc"]))
        if c["cache"] in TOP:
            K = K.view(TORCH[c["cache"]]).double() * t["Ks"][ids].double()[..., None]
            V = V.view(TORCH[c["cache"]]).double() * t["Vs"][ids].double()[..., None]
        K, V = (x.double().transpose(0, 1).flatten(1, 2)[:, since:n] for x in (K, V))
        q = t["Q"][b].double().unflatten(0, (c["Hk"], -1))
        z = (q @ K.transpose(1, 2).contiguous()) / math.sqrt(c["D"])
        lse[b] = torch.logsumexp(z, -1).flatten()
        O[b] = (torch.softmax(z, -1) @ V.contiguous()).flatten(0, 1)
    return [O, lse]


def exact(c, seed):
    t = _inputs(c, seed)
    return {"qk": _exact_qk, "cache": _exact_cache, "decode": _exact_decode}[c["op"]](c, t)
