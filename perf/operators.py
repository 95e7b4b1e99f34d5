"""Workloads of the operators around the retention core: what a decoder layer
does to its queries and keys before the core (rotary positions), to its
residual stream after it (the norms before and after a block with its gate and
residual scale), and what generation does with the last row of logits (a draw
under temperature, top-k, top-p and min-p).

``run`` computes a case either from elementary torch operations (``own``
false) or through ``aceflow_b200.cuda_ops`` (``own`` true); both take the same
state from ``prepare``.  ``exact`` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# --------------------------------------------------------------------- cases
def _rotary(name, B, T, heads, dim, rot, layout, dtype, positions, start, packed, inverse, scaling, factor):
    return dict(name=name, op="rotary", B=B, T=T, heads=heads, dim=dim, rot=rot, layout=layout, dtype=dtype,
                positions=positions, start=start, packed=packed, inverse=inverse, scaling=scaling, factor=factor)


def _norm(name, rows, d, x, h, y, gate, post, scale, pre, alpha, train):
    return dict(name=name, op="norm", rows=rows, d=d, x=x, h=h, y=y, gate=gate, post=post, scale=scale, pre=pre,
                alpha=alpha, train=train)


def _sample(name, rows, vocab, dtype, mode, context, masked, shape):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, mode=mode, context=context,
                masked=masked, shape=shape)


def listed():
    return [
        # one decode step of 64 streams, q and k of 8 heads of 256 inside the packed fp32 projection
        _rotary("rotary decode", 64, 1, 16, 256, 256, "interleaved", "fp32", "random", 0, True, False, "none", 1.0),
        # the 8 x 4096 prompt of a d_model 2048 layer, q and k inside the packed bf16 projection
        _rotary("rotary prompt", 8, 4096, 16, 256, 256, "interleaved", "bf16", "start", 0, True, False, "none", 1.0),
        # the gradient through half of each head, frequencies by parts for 8 times the trained length
        _rotary("rotary gradient", 4, 2047, 9, 128, 64, "half", "fp32", "start", 0, False, True, "yarn", 8.0),
        # one 65536-token stream of a d_model 4096 layer that continues far behind its start
        _rotary("rotary long", 1, 65536, 32, 256, 256, "half", "bf16", "start", 1000003, True, False, "linear", 16.0),
        # the seam between two blocks at one token of 64 streams: fp32 residual stream, bf16 activations
        _norm("seam decode", 64, 2048, "fp32", "bf16", "bf16", False, True, False, True, 1.0, False),
        # the same over a prompt, with a gate and a learnt residual scale
        _norm("seam prompt", 32768, 2048, "bf16", "bf16", "bf16", True, True, True, True, 1.0, False),
        # a training step of the seam: outputs and all gradients
        _norm("seam training", 32768, 2048, "bf16", "bf16", "bf16", True, True, True, True, 1.0, True),
        # an odd width in fp32, with a scaled residual and no norm behind the block
        _norm("seam odd", 1021, 1531, "fp32", "fp32", "fp32", True, False, True, True, 2.2, True),
        # one stream of a 32000-token vocabulary with the engine's usual settings
        _sample("sample one", 1, 32000, "fp32", "usual", 60, False, "peaked"),
        # 64 streams, each with its own settings
        _sample("sample batch", 64, 32000, "fp32", "mixed", 60, False, "peaked"),
        # a full batch of a large vocabulary, a broad nucleus
        _sample("sample large", 256, 131072, "fp32", "nucleus", 0, False, "broad"),
        # an odd vocabulary in bf16 (many equal logits), masked tokens and a row with nothing left
        _sample("sample masked", 37, 50257, "bf16", "mixed", 0, True, "broad"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "norm", "norm", "sample", "sample"])
    if kind == "rotary":
        heads, dim = _log(rng, 1, 48), rng.choice([16, 40, 64, 96, 128, 192, 256])
        rot = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        tokens = _log(rng, 1, min(200000, (1 << 27) // (heads * dim)))
        B = _log(rng, 1, min(tokens, 64))
        packed = heads % 2 == 0 and rng.random() < 0.5
        scaling = rng.choice(["none", "linear", "yarn"])
        c = _rotary("", B, max(1, tokens // B), heads, dim, rot, rng.choice(["interleaved", "half"]),
                    rng.choice(["fp32", "bf16"]), rng.choice(["start", "random"]), rng.choice([0, 17, 4096, 2000001]),
                    packed, rng.random() < 0.4, scaling, 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]))
    elif kind == "norm":
        d = _log(rng, 64, 8192) if rng.random() < 0.5 else 64 * _log(rng, 1, 128)
        rows = _log(rng, 1, max(1, min(65536, (1 << 25) // d)))
        gate, post, scale, pre = (rng.random() < 0.6 for _ in range(4))
        c = _norm("", rows, d, rng.choice(["fp32", "bf16"]), rng.choice(["fp32", "bf16"]),
                  rng.choice(["fp32", "bf16"]), gate, post, scale, pre or not post, rng.choice([1.0, 1.7]),
                  rng.random() < 0.5)
    else:
        vocab = _log(rng, 100, 200000)
        rows = _log(rng, 1, max(1, min(512, (1 << 24) // vocab)))
        c = _sample("", rows, vocab, rng.choice(["fp32", "bf16"]), rng.choice(["usual", "mixed", "nucleus", "plain"]),
                    rng.choice([0, 0, 7, 60]), rng.random() < 0.3, rng.choice(["peaked", "broad"]))
    del c["name"]
    return c


# -------------------------------------------------------------------- inputs
def _frequencies(c):
    """Rotation frequencies of a case (fp32 values, held on the host in 64
    bits while they are made) and the factor on the rotated values."""
    half, base, s = c["rot"] // 2, 10000.0, c["factor"]
    i = torch.arange(half, dtype=torch.float64)
    f = base ** (-i / half)
    if c["scaling"] == "linear":
        return f / s, 1.0
    if c["scaling"] == "yarn":
        length = 4096.0
        turns = length * f / (2 * math.pi)  # full turns within the trained length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / s * (1.0 - keep), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _prepare_rotary(c, g, dev):
    B, T, heads, dim, dt = c["B"], c["T"], c["heads"], c["dim"], DTYPES[c["dtype"]]
    width = heads * dim
    row = width + width // 2 if c["packed"] else width  # q | k | v per token, or the rotated heads alone
    x = torch.empty(B, T, row, dtype=dt, device=dev).normal_(generator=g)
    x = x[..., :width].unflatten(-1, (heads, dim))
    f, scale = _frequencies(c)
    pos = c["start"]
    if c["positions"] == "random":  # streams of different lengths so far
        pos = torch.randint(0, 32768, (B, T), generator=g, device=dev, dtype=torch.int32) + c["start"]
    return dict(x=x, inv_freq=f.float().to(dev), scale=scale, positions=pos)


def _prepare_norm(c, g, dev):
    rows, d = c["rows"], c["d"]

    def make(kind, s=1.0):
        return torch.empty(rows, d, dtype=DTYPES[c[kind]], device=dev).normal_(0, s, generator=g)

    def weight(on, mean, s):
        return torch.empty(d, device=dev).normal_(mean, s, generator=g) if on else None

    st = dict(x=make("x", 2.0), h=make("h", 0.7), gate=make("h", 1.5) if c["gate"] else None,
              post_w=weight(c["post"], 1.0, 0.1), scale=weight(c["scale"], 0.3, 0.05), pre_w=weight(c["pre"], 1.0, 0.1))
    if c["train"]:
        st["dz"], st["dy"] = make("x", 0.1), make("y", 0.1) if c["pre"] else None
    return st


def _prepare_sample(c, g, dev):
    rows, V = c["rows"], c["vocab"]
    sd, lift = (2.0, 9.0) if c["shape"] == "peaked" else (2.5, 3.0)
    lg = torch.empty(rows, V, device=dev).normal_(0, sd, generator=g)
    few = min(V, 40)  # the continuations the context asks for
    ids = torch.randint(0, V, (rows, few), generator=g, device=dev)
    lg.scatter_(1, ids, lift + 2.0 * torch.randn(rows, few, generator=g, device=dev))
    if c["masked"]:  # tokens a grammar forbids; one row forbids everything
        lg.masked_fill_(torch.rand(rows, V, generator=g, device=dev) < 0.3, -math.inf)
        lg[rows // 2].fill_(-math.inf)
    st = dict(logits=lg.to(DTYPES[c["dtype"]]), uniforms=torch.rand(rows, generator=g, device=dev), context=None,
              penalty=1.0)
    if c["context"]:
        ctx = torch.randint(0, V, (rows, c["context"]), generator=g, device=dev, dtype=torch.int32)
        ctx[:, : c["context"] // 3] = ids[:, :1].int()
        ctx[:, -1] = -1
        st["context"], st["penalty"] = ctx, 1.2
    mode = c["mode"]
    if mode == "usual":  # generate_stream's defaults and a min-p floor
        st.update(temperature=0.7, top_k=40, top_p=0.9, min_p=0.02)
    elif mode == "nucleus":
        st.update(temperature=1.0, top_k=0, top_p=0.95, min_p=0.0)
    elif mode == "plain":
        st.update(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    else:  # every stream its own settings, a greedy one among them
        def pick(values, dt):
            i = torch.randint(0, len(values), (rows,), generator=g, device=dev)
            return torch.tensor(values, dtype=dt, device=dev)[i]

        st.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32),
                  top_k=pick([0, 0, 1, 20, 50, 1000], torch.int32),
                  top_p=pick([1.0, 0.98, 0.95, 0.9, 0.5], torch.float32),
                  min_p=pick([0.0, 0.0, 0.01, 0.1], torch.float32))
    return st


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    st = {"rotary": _prepare_rotary, "norm": _prepare_norm, "sample": _prepare_sample}[case["op"]](case, g, dev)
    st["case"] = dict(case)
    return st


# ------------------------------------------------------------ rotary positions
def _rotary_plain(c, st):
    x, rot = st["x"], c["rot"]
    pos = st["positions"]
    if not torch.is_tensor(pos):
        pos = (pos + torch.arange(c["T"], device=x.device)).expand(c["B"], c["T"])
    angle = pos.double()[..., None] * st["inv_freq"].double()  # [B, T, rot / 2]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    cos, sin = st["scale"] * cos, st["scale"] * (-sin if c["inverse"] else sin)
    xf = x.float()
    if c["layout"] == "interleaved":
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
    else:
        a, b = xf[..., : rot // 2], xf[..., rot // 2: rot]
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((u, v), -1)
    return torch.cat((turned, xf[..., rot:]), -1).to(x.dtype)


def _rotary_exact(c, st):
    x, half = st["x"].double(), c["rot"] // 2
    B, T, f = c["B"], c["T"], st["inv_freq"].double()
    if torch.is_tensor(st["positions"]):
        p = st["positions"].double()
    else:
        p = torch.arange(T, device=x.device, dtype=torch.float64).repeat(B, 1) + float(st["positions"])
    phase = torch.polar(torch.full((B, T, half), st["scale"], dtype=torch.float64, device=x.device),
                        p.unsqueeze(-1) * f * (-1.0 if c["inverse"] else 1.0)).unsqueeze(2)
    out = x.clone()
    first = slice(0, 2 * half, 2) if c["layout"] == "interleaved" else slice(0, half)
    second = slice(1, 2 * half, 2) if c["layout"] == "interleaved" else slice(half, 2 * half)
    z = torch.complex(x[..., first], x[..., second]) * phase
    out[..., first], out[..., second] = z.real, z.imag
    return out


# ------------------------------------------------- the seam between two blocks
EPS = 1e-6


def _seam_plain(c, st):
    x, h = st["x"].float(), st["h"].float()
    r1 = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) if c["post"] else None
    n = h * r1 * st["post_w"] if c["post"] else h
    g = st["gate"].float() if c["gate"] else None
    sig = 1.0 / (1.0 + torch.exp(-g)) if c["gate"] else None
    m = n * (g * sig) if c["gate"] else n
    m = m * st["scale"] if c["scale"] else m
    z = c["alpha"] * x + m
    out = {"z": z.to(DTYPES[c["x"]])}
    r2 = torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) if c["pre"] else None
    if c["pre"]:
        out["y"] = (z * r2 * st["pre_w"]).to(DTYPES[c["y"]])
    if not c["train"]:
        return out
    dz = st["dz"].float()
    if c["pre"]:
        dy, zh = st["dy"].float(), z * r2
        out["dpre_w"] = (dy * zh).sum(0)
        t = dy * st["pre_w"]
        dz = dz + r2 * (t - zh * (t * zh).mean(-1, keepdim=True))
    out["dx"] = (c["alpha"] * dz).to(DTYPES[c["x"]])
    swish = g * sig if c["gate"] else 1.0
    s = st["scale"] if c["scale"] else 1.0
    if c["scale"]:
        out["dscale"] = (dz * swish * n).sum(0)
    if c["gate"]:
        out["dgate"] = (dz * s * n * (sig * (1.0 + g * (1.0 - sig)))).to(DTYPES[c["h"]])
    dn = dz * s * swish
    if c["post"]:
        hh = h * r1
        out["dpost_w"] = (dn * hh).sum(0)
        t = dn * st["post_w"]
        dn = r1 * (t - hh * (t * hh).mean(-1, keepdim=True))
    out["dh"] = dn.to(DTYPES[c["h"]])
    return out


def _seam_exact(c, st):
    """The definition in 64 bits; gradients by automatic differentiation."""
    leaf = {k: v.double().requires_grad_(c["train"]) for k, v in st.items()
            if torch.is_tensor(v) and k not in ("dz", "dy")}

    def normed(v, w):
        return v / torch.sqrt(v.square().sum(-1, keepdim=True) / c["d"] + EPS) * w

    block = normed(leaf["h"], leaf["post_w"]) if c["post"] else leaf["h"]
    if c["gate"]:
        block = leaf["gate"] * torch.sigmoid(leaf["gate"]) * block
    if c["scale"]:
        block = leaf["scale"] * block
    z = leaf["x"] * c["alpha"] + block
    out = {"z": z}
    if c["pre"]:
        out["y"] = normed(z, leaf["pre_w"])
    if c["train"]:
        loss = (z * st["dz"].double()).sum()
        if c["pre"]:
            loss = loss + (out["y"] * st["dy"].double()).sum()
        for k, v in zip(leaf, torch.autograd.grad(loss, list(leaf.values()))):
            out["d" + k] = v
    return {k: v.detach() for k, v in out.items()}


def _seam_own(c, st):
    from aceflow_b200 import cuda_ops

    kw = dict(gate=st["gate"], post_w=st["post_w"], scale=st["scale"], pre_w=st["pre_w"], alpha=c["alpha"])
    if not c["train"]:
        z, y = cuda_ops.residual_norm(st["x"], st["h"], eps=EPS, out_dtype=DTYPES[c["y"]], **kw)
        return {"z": z, "y": y} if c["pre"] else {"z": z}
    z, y, stats = cuda_ops.residual_norm(st["x"], st["h"], eps=EPS, out_dtype=DTYPES[c["y"]], want_stats=True, **kw)
    g = cuda_ops.residual_norm_backward(st["dz"], st["dy"], st["x"], st["h"], stats, **kw)
    out = {"z": z, "y": y, "dx": g.x, "dh": g.h, "dgate": g.gate, "dpost_w": g.post_w, "dscale": g.scale,
           "dpre_w": g.pre_w}
    return {k: v for k, v in out.items() if v is not None}


# ------------------------------------------------------------------ the draw
def _column(v, rows, dt, dev):
    """A setting as one value per row (a number stands for all rows)."""
    return (v.to(dt) if torch.is_tensor(v) else torch.full((rows,), v, dtype=dt, device=dev))[:, None]


def _sample_plain(c, st):
    lg, dev = st["logits"].float(), st["logits"].device
    rows, V = lg.shape
    if st["context"] is not None:
        seen = torch.zeros(rows, V + 1, dtype=torch.bool, device=dev)
        ids = st["context"].long()
        seen.scatter_(1, torch.where((ids >= 0) & (ids < V), ids, V), True)
        pen = _column(st["penalty"], rows, torch.float32, dev)
        lg = torch.where(seen[:, :V], torch.where(lg > 0, lg / pen, lg * pen), lg)
    lg = torch.where(lg == lg, lg, -math.inf)
    t = _column(st["temperature"], rows, torch.float64, dev)
    k = _column(st["top_k"], rows, torch.int64, dev)
    p = _column(st["top_p"], rows, torch.float32, dev).double()
    floor = _column(st["min_p"], rows, torch.float32, dev).double()
    t = t.float().double()
    val, ids = torch.sort(lg, dim=1, descending=True, stable=True)
    top = val[:, :1].double()
    w = torch.exp((val.double() - top) / t.clamp_min(1e-5))  # which token a border falls on: 64 bits
    w = torch.where(val == -math.inf, 0.0, w)
    place = torch.arange(V, device=dev)[None]
    keep = (place < torch.where(k > 0, k, V)) & (w > 0)
    w = torch.where(keep, w, 0.0)
    run_sum = w.cumsum(1)
    before = run_sum - w
    z = run_sum[:, -1:]
    keep &= (before <= p.clamp_min(0.0) * z) | (p >= 1.0)  # through the first item that crosses top_p
    keep &= w >= floor.clamp(0.0, 1.0)
    last = keep.sum(1, keepdim=True) - 1
    mass = run_sum.gather(1, last.clamp_min(0))
    target = st["uniforms"].double()[:, None] * mass
    at = torch.minimum((run_sum < target).sum(1, keepdim=True), last.clamp_min(0))
    greedy = ~(t > 1e-4)
    at = torch.where(greedy, 0, at)
    token = ids.gather(1, at)
    logp = torch.where(greedy, 0.0, torch.log(w.gather(1, at)) - torch.log(mass))
    empty = top == -math.inf
    token, logp = torch.where(empty, -1, token), torch.where(empty, -math.inf, logp)
    return {"token": token[:, 0].int(), "logprob": logp[:, 0].float()}


def _sample_exact(c, st):
    """Row by row on the host, in 64 bits: the log-probability of the token
    that the definition draws (the token itself is a whole number)."""
    import numpy as np

    def setting(name, r):
        v = st[name]
        return float(v[r]) if torch.is_tensor(v) else float(np.float32(v))

    lg = st["logits"].float().cpu().numpy()
    u = st["uniforms"].cpu().numpy().astype(np.float64)
    ctx = None if st["context"] is None else st["context"].cpu().numpy()
    rows, V = lg.shape
    out = np.zeros(rows)
    for r in range(rows):
        row = lg[r].copy()
        if ctx is not None:
            seen = np.unique(ctx[r][(ctx[r] >= 0) & (ctx[r] < V)])
            pen = np.float32(st["penalty"])
            row[seen] = np.where(row[seen] > 0, row[seen] / pen, row[seen] * pen)
        t = setting("temperature", r)
        if not np.any(row > -np.inf):
            out[r] = -np.inf
            continue
        if t <= 1e-4:
            continue
        live = np.flatnonzero(row > -np.inf)
        order = live[np.lexsort((live, -row[live].astype(np.float64)))]
        k = int(setting("top_k", r))
        order = order[:k] if k > 0 else order
        x = (row[order].astype(np.float64) - float(row[order[0]])) / t
        q = np.exp(x) / float(np.exp(x).sum(dtype=np.longdouble))
        if setting("top_p", r) < 1.0:
            q = q[: 1 + int(np.searchsorted(np.cumsum(q), setting("top_p", r), side="right"))]
        q = q[q >= min(setting("min_p", r), 1.0) * q[0]]
        c_sum = np.cumsum(q)
        i = min(int(np.searchsorted(c_sum, u[r] * c_sum[-1], side="left")), len(q) - 1)
        out[r] = math.log(q[i] / c_sum[-1])
    return {"token": None, "logprob": torch.from_numpy(out)}


def _sample_own(c, st):
    from aceflow_b200 import cuda_ops

    token, logp = cuda_ops.sample_tokens(st["logits"], st["uniforms"], temperature=st["temperature"],
                                         top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"],
                                         repetition_penalty=st["penalty"], context=st["context"],
                                         return_logprobs=True)
    return {"token": token, "logprob": logp}


# ------------------------------------------------------------------------ run
def run(state):
    c = state["case"]
    if c["op"] == "rotary":
        if own:
            from aceflow_b200 import cuda_ops

            return cuda_ops.rotary(state["x"], state["inv_freq"], state["positions"], layout=c["layout"],
                                   scale=state["scale"], inverse=c["inverse"])
        return _rotary_plain(c, state)
    if c["op"] == "norm":
        return _seam_own(c, state) if own else _seam_plain(c, state)
    return _sample_own(c, state) if own else _sample_plain(c, state)


def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _rotary_exact, "norm": _seam_exact, "sample": _sample_exact}[case["op"]](case, st)


def work(case):
    size = {"fp32": 4, "bf16": 2}
    c = case
    if c["op"] == "rotary":
        n = c["B"] * c["T"] * c["heads"] * c["dim"]
        pos = 4 * c["B"] * c["T"] if c["positions"] == "random" else 0
        turned = c["B"] * c["T"] * c["heads"] * c["rot"]
        return {"bytes": 2 * n * size[c["dtype"]] + pos + 2 * c["rot"], "flops": 4 * turned}
    if c["op"] == "norm":
        n, x, h, y = c["rows"] * c["d"], size[c["x"]], size[c["h"]], size[c["y"]]
        gate = h if c["gate"] else 0
        y = y if c["pre"] else 0
        weights = 4 * c["d"] * (c["post"] + c["scale"] + c["pre"])
        b = n * (x + h + gate + x + y) + weights  # forward: x, h, gate in; z, y out
        f = n * 12
        if c["train"]:  # and dz, dy in; dx, dh, dgate and the weights' gradients out
            b += n * (x + y + x + h + gate) + weights
            f += n * 30
        return {"bytes": b, "flops": f}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * size[c["dtype"]] + c["rows"] * (12 + 4 * c["context"]), "flops": 6 * n}
