"""The pieces of a trainable attention block in the conv layout ([B, C, T], time contiguous) as they are measured:

  norm    LayerNorm over the channels, forward, and forward + backward with the gradients of its affine pair
  bias    the learned relative-position bias by buckets as a [H, Tq, Tk] tensor, with the gradient of its table
  attend  attention with that bias inside: training (all gradients), whole prompts, and one new token over a cache

`own` False computes them from elementary torch operations in 32 bits, `own` True through neuralsvb_amd.functional."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------------
def _norm(dtype, train, b, c, t, affine="float32"):
    return {"op": "norm", "dtype": dtype, "train": train, "b": b, "c": c, "t": t, "affine": affine}


def _bias(dtype, h, tq, tk, n=32, far=128, both=True):
    return {"op": "bias", "dtype": dtype, "h": h, "tq": tq, "tk": tk, "n": n, "far": far, "both": both}


def _attend(dtype, train, b, h, kv, dk, tq, tk, causal=False, both=True, ragged=True, n=32, far=128):
    return {"op": "attend", "dtype": dtype, "train": train, "b": b, "h": h, "kv": kv, "dk": dk, "tq": tq, "tk": tk,
            "causal": causal, "both": both, "ragged": ragged, "n": n, "far": far}


def listed():
    return [
        # a batch of decoders that each normalise one new frame: nothing but launch latency
        {"name": "norm_token", **_norm("float32", False, 8, 256, 1)},
        # the content encoder's width and length over a training batch of 16 clip pairs
        {"name": "norm_train", **_norm("float32", True, 32, 256, 562)},
        # the same block at the full mel length in half the bytes, odd row pitch
        {"name": "norm_train_bf16", **_norm("bfloat16", True, 16, 384, 1125)},
        # a wide model's batch: memory traffic alone
        {"name": "norm_wide_bf16", **_norm("bfloat16", True, 32, 1024, 2048, "bfloat16")},
        # the bias of the content encoder's four heads as a tensor, for a caller that makes its own scores
        {"name": "bias_encoder", **_bias("float32", 4, 562, 562)},
        # a long prompt's bias, causal buckets
        {"name": "bias_long", **_bias("float32", 8, 2048, 2051, 64, 512, False)},
        # training the content encoder: 4 heads of 64, padded clips, exact arithmetic
        {"name": "train_encoder", **_attend("float32", True, 32, 4, 4, 64, 562, 562)},
        # the same in bf16 on short odd clips, head width between the tile sizes
        {"name": "train_short_bf16", **_attend("bfloat16", True, 24, 4, 4, 48, 211, 211)},
        # training a causal decoder with shared key / value heads on long sequences
        {"name": "train_causal_bf16", **_attend("bfloat16", True, 2, 16, 4, 128, 2048, 2048, True, False, False)},
        # a prompt, forward only
        {"name": "prompt_bf16", **_attend("bfloat16", False, 2, 8, 8, 64, 2000, 2000, True, False, False)},
        # one new token for each of 16 requests over caches of different lengths, shared heads
        {"name": "token_cache_bf16", **_attend("bfloat16", False, 16, 16, 4, 64, 1, 8192, True, False)},
        # one new token of one short request
        {"name": "token_short", **_attend("float32", False, 1, 4, 4, 64, 1, 130, True, False)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16"])
    what = rng.choice(["norm", "bias", "train", "train", "prompt", "token"])
    both = rng.random() < 0.5
    n, far = rng.choice([(8, 20), (16, 64), (32, 128), (64, 512)])
    if what == "norm":
        c, t = _log(rng, 16, 1024), _log(rng, 1, 2048)
        return _norm(dtype, rng.random() < 0.75, max(1, min(_log(rng, 1, 64), (1 << 25) // (c * t))), c, t,
                     rng.choice(["float32", dtype]))
    if what == "bias":
        return _bias(dtype, rng.randint(1, 8), _log(rng, 1, 2048), _log(rng, 1, 2048), n, far, both)
    kv, dk = rng.choice([1, 2, 4]), rng.choice([16, 32, 48, 64, 80, 96, 128])
    h = kv * rng.choice([1, 1, 2, 4])
    causal = rng.random() < 0.5
    if what == "token":
        tk = _log(rng, 1, 8192)
        return _attend(dtype, False, _log(rng, 1, 16), h, kv, dk, 1, tk, True, False, True, n, far)
    t = _log(rng, 1, 2048)
    b = max(1, min(_log(rng, 1, 32), int(2e10 // (h * dk * t * t * (3 if dtype == "float32" else 1)))))
    return _attend(dtype, what == "train", b, h, kv, dk, t, t, causal, both and not causal, rng.random() < 0.5, n, far)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=dev) * std + mean).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        b, c, t = case["b"], case["c"], case["t"]
        adt = DTYPES[case["affine"]]
        s["x"] = normal(b, c, t, std=2.0, mean=0.5)
        s["gamma"], s["beta"] = normal(c, std=0.2, mean=1.0, dtype=adt), normal(c, std=0.2, dtype=adt)
        s["dy"] = normal(b, c, t)
        leaves = ("x", "gamma", "beta")
    elif case["op"] == "bias":
        s["table"] = normal(case["n"], case["h"], std=0.5)
        s["dy"] = normal(case["h"], case["tq"], case["tk"])
        leaves = ("table",)
    else:
        b, h, kv, dk, tq, tk = (case[m] for m in ("b", "h", "kv", "dk", "tq", "tk"))
        if tq == tk:                                                     # one projection's output, cut by channels
            y = normal(b, (h + 2 * kv) * dk, tk)
            s["q"], s["k"], s["v"] = y[:, :h * dk], y[:, h * dk:(h + kv) * dk], y[:, (h + kv) * dk:]
        else:                                                            # new tokens, and a cache
            s["q"], s["k"], s["v"] = normal(b, h * dk, tq), normal(b, kv * dk, tk), normal(b, kv * dk, tk)
        s["table"] = normal(case["n"], h, std=0.5, dtype=torch.float32)
        s["dy"] = normal(b, h * dk, tq)
        s["keep"] = s["q_start"] = None
        if case["ragged"]:
            length = torch.randint((tk + 1) // 2, tk + 1, (b,), generator=gen, device=dev)
            if tq == tk:
                s["keep"] = (torch.arange(tk, device=dev)[None] < length[:, None]).float()
            else:
                s["q_start"] = (length - tq).int()
        leaves = ("q", "k", "v", "table")
    if case.get("train", True):
        s["leaves"] = tuple(s[m].detach().requires_grad_() for m in leaves)
        s.update(zip(leaves, s["leaves"]))
    return s


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "norm":
        n = case["b"] * case["c"] * case["t"]
        return {"bytes": n * size * (5 if case["train"] else 2), "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "bias":
        n = case["h"] * case["tq"] * case["tk"]
        return {"bytes": 2 * n * size, "flops": n}
    b, h, kv, dk, tq, tk = (case[m] for m in ("b", "h", "kv", "dk", "tq", "tk"))
    seen = 0.75 if case["ragged"] else 1.0                               # the keys that the mean request holds
    pairs = b * h * tq * tk * seen * (0.5 if case["causal"] and tq == tk else 1.0)
    once = b * (2 * h * dk * tq + 2 * kv * dk * tk * seen) * size        # q, out; k, v
    if case["train"]:                                                    # again: dq, dout; dk, dv
        return {"bytes": 2 * once, "flops": 14 * pairs * dk}
    return {"bytes": once, "flops": 4 * pairs * dk}


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _bucket(rel, n, far, both):
    """Bucket of the key at distance `rel` behind (> 0) or before (< 0) the query: one for each near distance, then
    logarithmically wider ones up to `far`, and one for all that is further."""
    if both:
        n //= 2
        base, m = (rel > 0).long() * n, rel.abs()
    else:
        base, m = torch.zeros_like(rel), (-rel).clamp(min=0)
    near = n // 2
    wide = torch.log(m.clamp(min=1).double() / near) / math.log(far / near) * (n - near)
    wide = (near + torch.floor(wide + 1e-9).long()).clamp(max=n - 1)     # (1e-9: a border belongs to the further bucket)
    return base + torch.where(m < near, m, wide)


def _by_bucket(d, bucket, n):
    """Sums of d [H, Tq, Tk] over its diagonals, then over the diagonals of a bucket -> [n, H].  bucket [Tq + Tk - 1]: of the
    diagonal key - query = index - (Tq - 1)."""
    h, tq, tk = d.shape
    skew = torch.cat([d.flip(1), d.new_zeros(h, tq, tq)], 2).reshape(h, -1)[:, :tq * (tq + tk - 1)]
    sums = skew.reshape(h, tq, tq + tk - 1).double().sum(1)              # row i moved right by its distance from the last row
    return torch.zeros(n, h, dtype=torch.float64, device=d.device).index_add_(0, bucket, sums.t().contiguous())


def _plain_norm(s):
    x, g, b = s["x"].detach().float(), s["gamma"].detach().float()[:, None], s["beta"].detach().float()[:, None]
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    xh = (x - mean) * rstd
    y = (xh * g + b).to(s["x"].dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gy = dy * g
    dx = rstd * (gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(y.dtype), "dgamma": (dy * xh).sum((0, 2)).to(s["gamma"].dtype),
            "dbeta": dy.sum((0, 2)).to(s["beta"].dtype)}


def _plain_bias(s):
    tq, tk, n = s["tq"], s["tk"], s["n"]
    t = s["table"].detach()
    at = torch.arange(tk, device=t.device)[None] - torch.arange(tk - tq, tk, device=t.device)[:, None]
    bias = t[_bucket(at, n, s["far"], s["both"])].permute(2, 0, 1).contiguous()
    diagonals = _bucket(torch.arange(tq + tk - 1, device=t.device) - (tk - 1), n, s["far"], s["both"])
    return {"bias": bias, "dtable": _by_bucket(s["dy"].float(), diagonals, n).to(t.dtype)}


def _plain_attend(s):
    b, h, kv, dk, tq, tk, n = (s[m] for m in ("b", "h", "kv", "dk", "tq", "tk", "n"))
    g, dt, dev = h // kv, s["q"].dtype, s["q"].device
    q = s["q"].detach().float().reshape(b, kv, g, dk, tq)
    k, v = (s[m].detach().float().reshape(b, kv, 1, dk, tk) for m in ("k", "v"))
    table, scale = s["table"].detach().float(), dk ** -0.5
    start = torch.full((1,), tk - tq, device=dev) if s["q_start"] is None else s["q_start"].long()
    at = torch.arange(tk, device=dev)[None, None] - (start[:, None] + torch.arange(tq, device=dev))[:, :, None]
    bias = table[_bucket(at, n, s["far"], s["both"])].permute(0, 3, 1, 2).reshape(-1, kv, g, tq, tk)
    score = torch.matmul(q.transpose(-1, -2), k) * scale + bias
    hide = at > 0 if s["causal"] else torch.zeros_like(at, dtype=torch.bool)
    if s["keep"] is not None:
        hide = hide | (s["keep"] == 0)[:, None, :]
    score = score.masked_fill(hide[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))        # (a row without keys stays zero)
    out = torch.matmul(v, p.transpose(-1, -2)).reshape(b, h * dk, tq).to(dt)
    if not s["train"]:
        return {"out": out}
    do = s["dy"].float().reshape(b, kv, g, dk, tq)
    dp = torch.matmul(do.transpose(-1, -2), v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(k, ds.transpose(-1, -2)) * scale
    dkey = torch.matmul(q, ds).sum(2) * scale
    dv = torch.matmul(do, p).sum(2)
    diagonals = _bucket(torch.arange(tq + tk - 1, device=dev) - (tk - 1), n, s["far"], s["both"])
    dtable = _by_bucket(ds.sum(0).reshape(h, tq, tk), diagonals, n)
    return {"out": out, "dq": dq.reshape(b, h * dk, tq).to(dt), "dk": dkey.reshape(b, kv * dk, tk).to(dt),
            "dv": dv.reshape(b, kv * dk, tk).to(dt), "dtable": dtable.float()}


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _own(s):
    from neuralsvb_amd import functional as SF
    if s["op"] == "norm":
        y = SF.layer_norm_nct(s["x"], s["gamma"], s["beta"], 1e-5)
        names = ("y", "dx", "dgamma", "dbeta")
    else:
        buckets = SF.RelativeBuckets(s["n"], s["far"], s["both"])
        if s["op"] == "bias":
            y = SF.bucket_bias(s["table"], buckets, s["tq"], s["tk"])
            names = ("bias", "dtable")
        else:
            y = SF.bucket_attention(s["q"], s["k"], s["v"], s["table"], buckets, s["h"], keep=s["keep"],
                                    causal=s["causal"], q_start=s["q_start"])
            names = ("out", "dq", "dk", "dv", "dtable")
    if "leaves" not in s:
        return {names[0]: y}
    return dict(zip(names, (y.detach(),) + torch.autograd.grad(y, s["leaves"], s["dy"])))


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "bias": _plain_bias, "attend": _plain_attend}[state["op"]](state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _bucket_of(rel, n, far, both):
    """As a number, in whole numbers alone: the wide bucket of distance m is the last t with near (far / near)^(t / w) <= m."""
    base = 0
    if both:
        n //= 2
        base = n if rel > 0 else 0
        m = abs(rel)
    else:
        m = max(-rel, 0)
    near = n // 2
    if m < near:
        return base + m
    w, t = n - near, 0
    while t + 1 < w and far ** (t + 1) * near ** (w - t - 1) <= m ** w:
        t += 1
    return base + near + t


def _bucket_map(case, offsets):
    span = case["far"] + 1
    lut = [_bucket_of(r, case["n"], case["far"], case["both"]) for r in range(-span, span + 1)]
    return torch.tensor(lut, device=offsets.device)[offsets.clamp(-span, span) + span]


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda t: t.detach().double().requires_grad_()  # noqa: E731
    if case["op"] == "norm":
        x, g, b = wide(s["x"]), wide(s["gamma"]), wide(s["beta"])
        y = torch.nn.functional.layer_norm(x.transpose(1, 2), (case["c"],), g, b, 1e-5).transpose(1, 2)
        if not case["train"]:
            return {"y": y.detach()}
        dx, dg, db = torch.autograd.grad(y, (x, g, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dgamma": dg, "dbeta": db}
    n, tq, tk, h = case["n"], case["tq"], case["tk"], case["h"]
    dev = s["table"].device
    start = s.get("q_start")
    start = torch.tensor([tk - tq], device=dev) if start is None else start.long()
    rows = start[:, None] + torch.arange(tq, device=dev)[None]                                     # [B or 1, Tq]
    rel = torch.arange(tk, device=dev) - rows[..., None]
    where = _bucket_map(case, rel)
    table = s["table"].detach().double()
    bias = table.t()[:, where].transpose(0, 1).contiguous().requires_grad_()                       # [B or 1, H, Tq, Tk]

    def table_gradient(d):
        return torch.stack([(d * (where == k)[:, None]).sum((0, 2, 3)) for k in range(n)])

    if case["op"] == "bias":
        return {"bias": bias[0].detach(), "dtable": table_gradient(s["dy"].double()[None])}
    b, kv, dk = case["b"], case["kv"], case["dk"]
    q, k, v = wide(s["q"]), wide(s["k"]), wide(s["v"])
    spread = lambda t: t.reshape(b, kv, 1, dk, tk).expand(b, kv, h // kv, dk, tk).reshape(b, h, dk, tk)  # noqa: E731
    score = q.reshape(b, h, dk, tq).transpose(2, 3) @ spread(k) / math.sqrt(dk) + bias
    see = torch.ones_like(rel, dtype=torch.bool) if not case["causal"] else rel <= 0
    if s["keep"] is not None:
        see = see & (s["keep"] != 0)[:, None]
    see = see[:, None]
    p = torch.softmax(score.masked_fill(~see, -1e300), -1) * see         # (-1e300: nothing is left of a hidden key beside a seen one)
    out = (spread(v) @ p.transpose(2, 3)).reshape(b, h * dk, tq)
    if not case["train"]:
        return {"out": out.detach()}
    dq, dkey, dv, dbias = torch.autograd.grad(out, (q, k, v, bias), s["dy"].double())
    return {"out": out.detach(), "dq": dq, "dk": dkey, "dv": dv, "dtable": table_gradient(dbias)}
