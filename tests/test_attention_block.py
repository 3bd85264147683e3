"""LayerNorm over channels with its gradient, the learned relative-position bias by buckets, and attention with that bias inside,
against plain forms in 64 bits."""
import math

import pytest
import torch

from neuralsvb_amd import functional as SF

U32 = 2.0 ** -24                       # half a step of the type, relative to the value
UBF = 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_dt = pytest.mark.parametrize("dt", ["f32", "bf16"])


def near(got, want, tol, what, size=None):
    """2-norm of the difference against the 2-norm of the result (absolutely against 1 where the result is 0), or against `size`."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    off, size = float((got - want).norm()), float(want.norm()) if size is None else size
    assert off <= tol * (size if size else 1.0), f"{what}: {off / (size or 1.0):.3g} > {tol:.3g}"


# ---- plain forms -----------------------------------------------------------------------------------------------------
def bucket_of(o, n, far, both):
    base, m = 0, max(-o, 0)
    if both:
        n //= 2
        base, m = (n if o > 0 else 0), abs(o)
    near_ = n // 2
    if m < near_:
        return base + m
    t = 0
    while t + 1 < n - near_ and far ** (t + 1) * near_ ** (n - near_ - t - 1) <= m ** (n - near_):
        t += 1
    return base + near_ + t


def bucket_index(buckets, tq, tk, start):
    far = buckets.max_distance + 1
    lut = torch.tensor([bucket_of(o, buckets.n_buckets, buckets.max_distance, buckets.bidirectional) for o in range(-far, far + 1)])
    return lut[(torch.arange(tk)[None] - (start + torch.arange(tq)[:, None])).clamp(-far, far) + far]


def attention64(q, k, v, table, buckets, n_head, keep=None, causal=False, scale=None, q_start=None):
    """Everything in float64 with autograd, q [B, H dk, Tq] ... as the operator takes them."""
    B, D, tq = q.shape
    dk, tk = D // n_head, k.shape[2]
    g = n_head // (k.shape[1] // dk)
    starts = [tk - tq] * B if q_start is None else [int(s) for s in q_start] if isinstance(q_start, torch.Tensor) else [q_start] * B
    out = []
    for b in range(B):
        see = torch.ones(tq, tk, dtype=torch.bool)
        if keep is not None:
            see = see & (keep[b].cpu() != 0)
        if causal:
            see = see & (torch.arange(tk)[None] <= starts[b] + torch.arange(tq)[:, None])
        idx = bucket_index(buckets, tq, tk, starts[b])
        kept = see.any(0)                                                # (a key that nobody sees: whatever it holds)
        for h in range(n_head):
            qh = q[b, h * dk:(h + 1) * dk]
            kh = torch.where(kept, k[b, h // g * dk:(h // g + 1) * dk], torch.zeros(()).double())
            vh = torch.where(kept, v[b, h // g * dk:(h // g + 1) * dk], torch.zeros(()).double())
            s = qh.t() @ kh * (dk ** -0.5 if scale is None else scale) + table[:, h][idx]
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            e = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)).detach())
            total = e.sum(1, keepdim=True)
            out.append(vh @ (e / torch.where(total > 0, total, torch.ones_like(total))).t())
    return torch.cat(out).reshape(B, D, tq)


def leaves64(*ts):
    return [t.detach().double().cpu().requires_grad_() for t in ts]


# ---- LayerNorm over channels -----------------------------------------------------------------------------------------
# shapes: one position, shorter and longer than a tile, odd row pitches, one channel, more channels than rows of a pass, the widest
# register form, and beyond it
LN_SHAPES = [(1, 1, 1), (3, 7, 1), (2, 80, 5), (2, 130, 9), (2, 40, 33), (1, 256, 67), (2, 300, 131), (1, 700, 18), (1, 1030, 35)]


@_dt
@pytest.mark.parametrize("shape", LN_SHAPES)
def test_layer_norm_nct(dev, dt, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    B, C, T = shape
    x = (torch.randn(shape, generator=gen) * 2 + 0.5).to(DT[dt])
    gamma, beta = torch.randn(C, generator=gen) * 0.2 + 1, torch.randn(C, generator=gen)
    dy = torch.randn(shape, generator=gen).to(DT[dt])
    lx, lg, lb = leaves64(x, gamma, beta)
    want = torch.nn.functional.layer_norm(lx.transpose(1, 2), (C,), lg, lb, 1e-5).transpose(1, 2)
    want.backward(dy.double())
    dx, dg, db = (t.clone().to(dev).requires_grad_() for t in (x, gamma, beta))
    y = SF.layer_norm_nct(dx, dg, db)
    y.backward(dy.to(dev))
    # the sums over C and over B T positions have errors of at most (their number) half steps, of which random ones leave the root;
    # the result is rounded once to its type
    n = 8 * U32 * (math.sqrt(C) + 4)
    unit = UBF if dt == "bf16" else 0.0
    near(y, want.detach(), unit + n, "y")
    if C > 1:
        near(dg.grad, lg.grad, 8 * U32 * (math.sqrt(C) + math.sqrt(B * T) + 4), "dgamma")
    else:
        assert not dg.grad.any()                                         # (one channel is its own mean)
    near(db.grad, lb.grad, 8 * U32 * (math.sqrt(B * T) + 4), "dbeta")
    if C > 1:
        near(dx.grad, lx.grad, unit + 4 * n, "dx")
    else:
        assert float(dx.grad.float().abs().max()) < 1e-2                 # (one channel: exactly 0 but for the rounding of dy gamma rstd)
    with torch.no_grad():
        near(SF.layer_norm_nct(dx, dg, db), want.detach(), unit + n, "y without gradients")


def test_layer_norm_nct_affine_choices(dev):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 24, 37, generator=gen)
    for dt in (torch.float32, torch.bfloat16):
        for gamma, beta in ((None, None), (torch.randn(24, generator=gen), None), (None, torch.randn(24, generator=gen))):
            for adt in {torch.float32, dt}:
                g, b = (None if t is None else t.detach().to(adt) for t in (gamma, beta))
                (lx,) = leaves64(x.to(dt))
                lg, lb = (None if t is None else leaves64(t)[0] for t in (g, b))
                want = torch.nn.functional.layer_norm(lx.transpose(1, 2), (24,), lg, lb, 1e-5).transpose(1, 2)
                want.sum().backward()
                dx = x.to(dt).to(dev).requires_grad_()
                dg, db = (None if t is None else t.detach().clone().to(dev).requires_grad_() for t in (g, b))
                y = SF.layer_norm_nct(dx, dg, db)
                y.sum().backward()
                near(y, want.detach(), (UBF if dt == torch.bfloat16 else 0) + 1e-6, "y")
                for d, l in ((dg, lg), (db, lb)):
                    if d is not None:
                        assert d.grad.dtype == adt
                        # (dy = 1: dgamma is a sum of 74 values near 1 in size that nearly cancel: absolute, half a step of each)
                        assert float((d.grad.double().cpu() - l.grad).abs().max()) <= 74 * 4 * (UBF if adt == torch.bfloat16 else U32)


def test_layer_norm_nct_offset_input(dev):
    """A mean 300 times the deviation: variances from centred values."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(1, 64, 40, generator=gen) + 300
    (lx,) = leaves64(x)
    want = torch.nn.functional.layer_norm(lx.transpose(1, 2), (64,), None, None, 1e-5).transpose(1, 2)
    y = SF.layer_norm_nct(x.to(dev).requires_grad_(), None, None)
    near(y, want.detach(), 300 * 4 * U32, "y")          # (the mean is off by at most a few half steps of 300, the deviation is 1)


def test_layer_norm_nct_refusals(dev):
    x = torch.zeros(2, 8, 4, device=dev, requires_grad=True)
    one = torch.ones(8, device=dev)
    with pytest.raises(ValueError):
        SF.layer_norm_nct(x[0], one, one)
    with pytest.raises(ValueError):
        SF.layer_norm_nct(x, one[:7], one)
    with pytest.raises(ValueError):
        SF.layer_norm_nct(x, one.bfloat16(), one.bfloat16())
    with pytest.raises(TypeError):
        SF.layer_norm_nct(x.half(), one, one)
    with pytest.raises(TypeError):
        SF.layer_norm_nct(x.bfloat16(), one, one.bfloat16())
    with torch.no_grad():
        assert SF.layer_norm_nct(torch.zeros(2, 8, 0, device=dev), one, one).shape == (2, 8, 0)


# ---- the bias by buckets -----------------------------------------------------------------------------------------------
KINDS = [(8, 20, True), (16, 64, False), (32, 128, True), (64, 512, False), (6, 9, True), (2, 3, False), (4, 2, True)]


@pytest.mark.parametrize("kind", KINDS)
def test_bucket_bias(dev, kind):
    gen = torch.Generator().manual_seed(kind[0])
    bk = SF.RelativeBuckets(*kind)
    for dt in (torch.float32, torch.bfloat16):
        for h, tq, tk, start in ((1, 1, 1, None), (3, 1, 70, None), (2, 5, 3, None), (2, 37, 41, 7), (1, 66, 131, -40), (1, 3, 9, 1000)):
            table = torch.randn(kind[0], h, generator=gen).to(dt)
            d = torch.randn(h, tq, tk, generator=gen).to(dt)
            idx = bucket_index(bk, tq, tk, tk - tq if start is None else start)
            want = torch.zeros(kind[0], h, dtype=torch.float64).index_add_(0, idx.reshape(-1), d.double().permute(1, 2, 0).reshape(-1, h))
            size = torch.zeros(kind[0], h, dtype=torch.float64).index_add_(0, idx.reshape(-1), d.double().abs().permute(1, 2, 0).reshape(-1, h))
            t = table.to(dev).requires_grad_()
            bias = SF.bucket_bias(t, bk, tq, tk, start)
            assert torch.equal(bias.detach().cpu(), table[idx].permute(2, 0, 1))
            bias.backward(d.to(dev))
            # each of the sums' few steps rounds by half a step of at most the sum of the sizes; one rounding to the table's type
            tol = size * 64 * U32 + want.abs() * (UBF if dt == torch.bfloat16 else 0)
            assert ((t.grad.double().cpu() - want).abs() <= tol + 1e-30).all()


def test_bucket_bias_across_tiles(dev):
    """More offsets than a workgroup takes, rows in several chunks, odd widths."""
    gen = torch.Generator().manual_seed(5)
    bk = SF.RelativeBuckets(32, 128, True)
    d = torch.randn(2, 50, 1201, generator=gen)
    idx = bucket_index(bk, 50, 1201, 600)
    want = torch.zeros(32, 2, dtype=torch.float64).index_add_(0, idx.reshape(-1), d.double().permute(1, 2, 0).reshape(-1, 2))
    t = torch.randn(32, 2, generator=gen).to(dev).requires_grad_()
    bias = SF.bucket_bias(t, bk, 50, 1201, 600)
    assert torch.equal(bias.detach().cpu(), t.detach().cpu()[idx].permute(2, 0, 1))
    bias.backward(d.to(dev))
    near(t.grad, want, 64 * U32, "dtable")


def test_bucket_borders():
    """Borders in whole numbers: with near = 8 and 8 geometric buckets up to 128 every second one starts at a power of two."""
    bk = SF.RelativeBuckets(32, 128, True)
    assert list(bk.c.edge[:bk.c.n_edge]) == [12, 16, 23, 32, 46, 64, 91]
    for n, far, both in KINDS:
        c = SF.RelativeBuckets(n, far, both).c
        for m in range(0, 3 * far):
            want = bucket_of(-m, n, far, both)
            got = m if m < c.near else c.near + sum(e <= m for e in c.edge[:c.n_edge])
            assert got == want, (n, far, both, m)


def test_bucket_refusals(dev):
    for bad in ((1, 8, False), (66, 128, True), (7, 20, True), (2, 20, True), (32, 8, True), (32, 4000, True)):
        with pytest.raises(ValueError):
            SF.RelativeBuckets(*bad)
    bk = SF.RelativeBuckets(8, 20)
    t = torch.zeros(8, 2, device=dev)
    with pytest.raises(ValueError):
        SF.bucket_bias(t[:7], bk, 3, 3)
    with pytest.raises(TypeError):
        SF.bucket_bias(t.half(), bk, 3, 3)
    with pytest.raises(ValueError):
        SF.bucket_bias(t, bk, -1, 3)
    assert SF.bucket_bias(t, bk, 0, 3).shape == (2, 0, 3)


# ---- attention with the bias inside --------------------------------------------------------------------------------------
def case(seed, dt, B, H, Hkv, dk, tq, tk, n=16, table_dt=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, m * dk, t, generator=gen).to(DT[dt]) for m, t in ((H, tq), (Hkv, tk), (Hkv, tk)))
    table = (torch.randn(n, H, generator=gen) * 0.7).to(table_dt)
    return q, k, v, table, torch.randn(B, H * dk, tq, generator=gen).to(DT[dt])


def compare(dev, dt, tensors, dout, buckets, n_head, keep=None, causal=False, scale=None, q_start=None, place=None, what=""):
    """The operator's output and gradients against attention64's.  place: how a tensor reaches the device (its strides)."""
    # Rounded values: the result itself (half a step), and the weights P and dS as operands, half a step each of values whose errors
    # are independent over the sum: a 2-norm of at most the result's when values are random.  Three times half a step, then.
    # fp32: three bf16 parts keep 2^-25 of each operand; scores of size 8 carry 8 half steps into the weights' exponents, the sums
    # (up to 128 channels and some hundred keys) a few more.
    tol = 3 * UBF if dt == "bf16" else 128 * U32
    # dtable is fp32 for either type, and a bucket's sum cancels; with bf16 tensors delta comes from the output before its rounding, with P
    # in parts of 2^-8 each (two of them leave 2^-16: the bound)
    tol_table = {"bf16": 8 * 2.0 ** -16, "f32": 128 * U32}[dt] + (UBF if tensors[3].dtype == torch.bfloat16 else 0)
    want_leaves = leaves64(*tensors)
    want = attention64(*want_leaves, buckets, n_head, keep, causal, scale, q_start)
    want.backward(dout.double())
    got_leaves = [t.detach().to(dev) for t in tensors]
    if place:
        got_leaves[:3] = [place(t) for t in got_leaves[:3]]
    got_leaves = [t.requires_grad_() for t in got_leaves]
    opt = dict(keep=None if keep is None else keep.to(dev), causal=causal, scale=scale,
               q_start=q_start.to(dev) if isinstance(q_start, torch.Tensor) else q_start)
    got = SF.bucket_attention(*got_leaves, buckets, n_head, **opt)
    got.backward(dout.to(dev))
    near(got, want.detach(), tol, what + " out")
    for name, g, w in zip(("dq", "dk", "dv"), got_leaves, want_leaves):
        near(g.grad, w.grad, tol, f"{what} {name}")
    # Where all pairs share one bucket the sum over it is exactly 0 (each query's dS sum to 0) and only the terms have a size: per query
    # sum_j |dS_ij| <= 2 max_j |dout_i . v_j|, random values of about |dout_i| each, so their roundings are against |dout|.
    terms, sums = float(dout.double().norm()), float(want_leaves[3].grad.norm())
    near(got_leaves[3].grad, want_leaves[3].grad, tol_table, what + " dtable", terms if sums < 1e-9 * terms else sums)
    with torch.no_grad():
        near(SF.bucket_attention(*got_leaves, buckets, n_head, **opt), want.detach(), tol, what + " out without gradients")
    return got, got_leaves


# (B, H, Hkv, dk, Tq, Tk): one of everything, lengths around the tile sizes 32 / 64 / 128, widths around 32 / 64 / 96 / 128, shared heads
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 2, 1, 7, 1, 2), (2, 2, 2, 32, 31, 33), (1, 2, 2, 33, 64, 64), (1, 1, 1, 64, 65, 63), (1, 4, 2, 20, 130, 129),
          (1, 1, 1, 96, 3, 70), (1, 2, 1, 97, 5, 200), (1, 1, 1, 128, 129, 40)]


@_dt
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(dev, dt, shape):
    B, H, Hkv, dk, tq, tk = shape
    *t, do = case(sum(shape), dt, *shape)
    compare(dev, dt, t, do, SF.RelativeBuckets(16, 40, True), H, what="both sides")
    *t, do = case(sum(shape) + 1, dt, *shape)
    compare(dev, dt, t, do, SF.RelativeBuckets(16, 24, False), H, causal=True, what="causal")


@_dt
def test_attention_masks(dev, dt):
    """Padded keys inside and at the end, a batch entry without any key, and NaN / infinities behind the mask."""
    *t, do = case(1, dt, 4, 2, 1, 24, 45, 70)
    keep = torch.ones(4, 70)
    keep[0, 50:] = 0
    keep[1, ::3] = 0
    keep[1, 0:34] = 0                                                    # (a whole tile of 32)
    keep[2] = 0
    for x in (t[1], t[2]):
        x[keep[:, None, :].expand_as(x) == 0] = float("nan")
        x[0, :, 60] = float("inf")
    bk = SF.RelativeBuckets(16, 24, True)
    for causal in (False, True):
        got, leaves = compare(dev, dt, t, do, bk, 2, keep=keep, causal=causal, what=f"causal={causal}")
        assert not got[2].any()
        for x in leaves[:3]:
            assert not x.grad[2].any()
        assert not leaves[1].grad[0, :, 50:].any() and not leaves[2].grad[0, :, 50:].any()


@_dt
def test_attention_positions(dev, dt):
    """Queries anywhere against the keys: before all of them (nobody sees a key), behind, one start per batch entry, a full table."""
    bk = SF.RelativeBuckets(16, 24, True)
    for q_start in (-200, -3, 500, torch.tensor([0, 40, -70], dtype=torch.int32)):
        for causal in (False, True):
            *t, do = case(7, dt, 3, 2, 2, 16, 37, 66)
            got, leaves = compare(dev, dt, t, do, bk, 2, causal=causal, q_start=q_start, what=f"{q_start} {causal}")
            if causal and q_start is not None and not isinstance(q_start, torch.Tensor) and q_start == -200:
                assert not got.any() and not any(x.grad.any() for x in leaves)
    *t, do = case(8, dt, 1, 1, 1, 16, 40, 40, n=64)
    compare(dev, dt, t, do, SF.RelativeBuckets(64, 1024, True), 1, what="64 buckets")
    *t, do = case(9, dt, 1, 3, 1, 16, 40, 40, n=2, table_dt=torch.bfloat16 if dt == "bf16" else torch.float32)
    compare(dev, dt, t, do, SF.RelativeBuckets(2, 2, False), 3, scale=0.5, what="two buckets")


@_dt
def test_attention_strides(dev, dt):
    """Slices of one projection, an expanded batch, time not innermost, a base that no vector load is aligned to."""
    bk = SF.RelativeBuckets(16, 40, True)
    *t, do = case(11, dt, 2, 2, 2, 24, 41, 41)
    y = torch.cat(t[:3], 1).to(dev)
    parts = iter((y[:, :48], y[:, 48:96], y[:, 96:]))
    compare(dev, dt, t, do, bk, 2, place=lambda x: next(parts).detach(), what="slices")

    def shifted(x):
        room = torch.full((x.shape[0], x.shape[1], x.shape[2] + 3), float("nan"), device=x.device, dtype=x.dtype)
        room[:, :, 1:-2] = x
        return room[:, :, 1:-2].detach()
    compare(dev, dt, t, do, bk, 2, place=shifted, what="shifted")
    compare(dev, dt, t, do, bk, 2, place=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2).detach(), what="time outside")
    *t, do = case(12, dt, 1, 2, 1, 24, 41, 41)
    leaf = t[1].to(dev).requires_grad_()
    both = SF.bucket_attention(t[0].to(dev).expand(2, -1, -1), leaf.expand(2, -1, -1), t[2].to(dev).expand(2, -1, -1), t[3].to(dev), bk, 2)
    one = SF.bucket_attention(t[0].to(dev), leaf, t[2].to(dev), t[3].to(dev), bk, 2)
    assert torch.equal(both[0], one[0]) and torch.equal(both[1], one[0])
    twice = torch.autograd.grad(both, leaf, do.to(dev).expand(2, -1, -1).contiguous())[0]
    once = torch.autograd.grad(one, leaf, do.to(dev))[0]
    near(twice, 2 * once.double().cpu(), UBF if dt == "bf16" else U32, "broadcast keys")


def test_attention_subsets_of_gradients(dev):
    """Only the wanted gradients, each as with all of them; the same bits from every call."""
    bk = SF.RelativeBuckets(16, 40, True)
    *t, do = case(13, "bf16", 1, 4, 2, 40, 70, 90)
    t, do = [x.to(dev) for x in t], do.to(dev)

    def grads(which):
        ls = [x.detach().requires_grad_(i in which) for i, x in enumerate(t)]
        out = SF.bucket_attention(*ls, bk, 4)
        return dict(zip(which, torch.autograd.grad(out, [ls[i] for i in which], do)))
    full = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (0, 1, 2, 3)):
        for i, g in grads(which).items():
            assert torch.equal(g, full[i])


def test_attention_gradient_by_differences(dev):
    """dout . d out along a random direction of all inputs, central differences of the fp32 operator."""
    *t, do = case(14, "f32", 2, 2, 1, 16, 21, 40)
    t, do = [x.to(dev) for x in t], do.to(dev)
    bk = SF.RelativeBuckets(16, 24, True)
    gen = torch.Generator().manual_seed(15)
    step = [torch.randn(x.shape, generator=gen).to(dev) for x in t]
    ls = [x.detach().requires_grad_() for x in t]
    grads = torch.autograd.grad(SF.bucket_attention(*ls, bk, 2), ls, do)
    along = sum(float((g.double() * s.double()).sum()) for g, s in zip(grads, step))
    e = 2.0 ** -9
    with torch.no_grad():
        up, down = (SF.bucket_attention(*[x + w * e * s for x, s in zip(t, step)], bk, 2) for w in (1, -1))
    diff = float(((up.double() - down.double()) * do.double()).sum()) / (2 * e)
    # third derivatives: e^2 / 6 of values of the size of the result's norm; roundings: 128 half steps of the output over 2 e
    size = float(do.double().norm() * up.double().norm())
    assert abs(diff - along) <= size * (8 * e * e + 128 * U32 / (2 * e) / math.sqrt(do.numel()))


def test_attention_refusals(dev):
    bk = SF.RelativeBuckets(8, 20)
    q, kv, t = torch.zeros(2, 32, 5, device=dev), torch.zeros(2, 16, 9, device=dev), torch.zeros(8, 2, device=dev)
    ok = SF.bucket_attention(q, kv, kv, t, bk, 2)
    assert ok.shape == (2, 32, 5)
    for bad in (dict(q=q[0]), dict(k=kv[:, :15]), dict(v=kv[:, :, :8]), dict(t=t[:, :1]), dict(t=t[:7]), dict(k=kv[:1], v=kv[:1]), dict(n=3),
                dict(n=0), dict(keep=torch.ones(2, 8, device=dev)), dict(q_start=torch.zeros(2, dtype=torch.int64, device=dev)),
                dict(q_start=torch.zeros(3, dtype=torch.int32, device=dev)),
                dict(q=torch.zeros(2, 129, 5, device=dev), k=torch.zeros(2, 129, 5, device=dev), v=torch.zeros(2, 129, 5, device=dev),
                     t=torch.zeros(8, 1, device=dev), n=1)):
        with pytest.raises(ValueError):
            SF.bucket_attention(bad.get("q", q), bad.get("k", kv), bad.get("v", kv), bad.get("t", t), bk, bad.get("n", 2),
                                keep=bad.get("keep"), q_start=bad.get("q_start"))
    for bad in (dict(q=q.bfloat16()), dict(q=q.half(), k=kv.half(), v=kv.half()), dict(t=t.half()), dict(keep=torch.ones(2, 9, device=dev).bool())):
        with pytest.raises(TypeError):
            SF.bucket_attention(bad.get("q", q), bad.get("k", kv), bad.get("v", bad.get("k", kv)), bad.get("t", t), bk, 2, keep=bad.get("keep"))
    # nothing to do
    assert SF.bucket_attention(q[:, :, :0], kv, kv, t, bk, 2).shape == (2, 32, 0)
    leaf = q.clone().requires_grad_()
    out = SF.bucket_attention(leaf, kv[:, :, :0], kv[:, :, :0], t, bk, 2)
    assert out.shape == (2, 32, 5) and not out.any()
    out.sum().backward()
    assert not leaf.grad.any()


def test_block_together(dev):
    """A pre-norm block as it is used: norm, one projection for q, k, v, attention, output projection, residual; all gradients."""
    gen = torch.Generator().manual_seed(21)
    B, D, T, H = 2, 32, 45, 2
    x = torch.randn(B, D, T, generator=gen)
    ws = [torch.randn(3 * D, D, generator=gen) * D ** -0.5, torch.randn(3 * D, generator=gen) * 0.1, torch.randn(D, D, generator=gen) * D ** -0.5]
    gamma, beta, table = torch.rand(D, generator=gen) + 0.5, torch.randn(D, generator=gen) * 0.1, torch.randn(16, H, generator=gen)
    keep = torch.ones(B, T)
    keep[1, 30:] = 0
    bk = SF.RelativeBuckets(16, 24, True)
    ls = [t.clone().to(dev).requires_grad_() for t in (x, *ws, gamma, beta, table)]
    y = SF.linear_nct(SF.layer_norm_nct(ls[0], ls[4], ls[5]), ls[1], ls[2])
    a = SF.bucket_attention(y[:, :D], y[:, D:2 * D], y[:, 2 * D:], ls[6], bk, H, keep=keep.to(dev))
    out = ls[0] + SF.linear_nct(a, ls[3])
    do = torch.randn(out.shape, generator=gen)
    out.backward(do.to(dev))
    lw = leaves64(x, *ws, gamma, beta, table)
    n = torch.nn.functional.layer_norm(lw[0].transpose(1, 2), (D,), lw[4], lw[5], 1e-5)
    y = (n @ lw[1].t() + lw[2]).transpose(1, 2)
    a = attention64(y[:, :D], y[:, D:2 * D], y[:, 2 * D:], lw[6], bk, H, keep)
    want = lw[0] + lw[3] @ a
    want.backward(do.double())
    near(out, want.detach(), 128 * U32, "out")
    for name, g, w in zip(("x", "w_qkv", "b_qkv", "w_out", "gamma", "beta", "table"), ls, lw):
        near(g.grad, w.grad, 4 * 128 * U32, name)                        # (four operators deep)


def test_bias_tensor_is_the_bias_inside(dev):
    """bucket_bias is what bucket_attention adds: equal scores leave the softmax of the bias alone."""
    bk = SF.RelativeBuckets(16, 24, True)
    table = torch.randn(16, 1, generator=torch.Generator().manual_seed(2)).to(dev)
    bias = SF.bucket_bias(table, bk, 6, 40)[0]
    v = torch.eye(40)[:32].reshape(1, 32, 40).to(dev)
    out = SF.bucket_attention(torch.zeros(1, 32, 6, device=dev), torch.zeros(1, 32, 40, device=dev), v, table, bk, 1)
    near(out[0], torch.softmax(bias.double().cpu(), 1)[:, :32].t(), 128 * U32, "weights")


# ---- forms, masks and limits ---------------------------------------------------------------------------------------------
# few query rows over a cache that several workgroups share: heads in one wave, widths of every padded form, one and several queries
@_dt
@pytest.mark.parametrize("shape", [(3, 4, 2, 20, 1, 700), (1, 6, 1, 97, 2, 300), (1, 2, 2, 64, 16, 300), (1, 8, 1, 33, 4, 65)])
def test_attention_cached_tokens(dev, dt, shape):
    """One start per request; behind it the cache holds anything; some cached keys hidden."""
    B, H, Hkv, dk, tq, tk = shape
    *t, do = case(sum(shape), dt, *shape)
    starts = torch.tensor([tk - tq, 66, 0][:B], dtype=torch.int32)
    for x in (t[1], t[2]):
        for b in range(B):
            x[b, :, int(starts[b]) + tq:] = float("nan")
    keep = torch.ones(B, tk)
    keep[:, 5:60:7] = 0
    keep[0, 200:290] = 0
    for mask in (None, keep):
        compare(dev, dt, t, do, SF.RelativeBuckets(16, 40, False), H, keep=mask, causal=True, q_start=starts, what=f"masked {mask is not None}")
    *t, do = case(sum(shape) + 1, dt, *shape)
    compare(dev, dt, t, do, SF.RelativeBuckets(16, 40, True), H, what="all keys")


# keys of a tile over two waves (bf16), steps of a key tile over workgroups (8 heads to one), rows of less than 4, lengths behind whole tiles
@_dt
@pytest.mark.parametrize("shape", [(1, 1, 1, 33, 70, 300), (1, 2, 1, 100, 65, 270), (1, 1, 1, 128, 40, 385), (1, 8, 1, 16, 130, 40), (1, 2, 1, 100, 2, 3),
                                   (2, 3, 1, 72, 64, 259)])
def test_attention_split_work(dev, dt, shape):
    B, H, Hkv, dk, tq, tk = shape
    *t, do = case(sum(shape), dt, *shape)
    keep = torch.ones(B, tk)
    keep[0, 60:200] = 0
    keep[0, tk - 1] = 0
    compare(dev, dt, t, do, SF.RelativeBuckets(16, 40, True), H, keep=keep, what="masked")
    compare(dev, dt, t, do, SF.RelativeBuckets(16, 40, False), H, causal=True, what="causal")


@_dt
def test_attention_widest_tables(dev, dt):
    """The furthest border with the widest heads: the most LDS that a call takes."""
    *t, do = case(31, dt, 1, 2, 1, 128, 50, 50, n=64)
    compare(dev, dt, t, do, SF.RelativeBuckets(64, 1024, True), 2, what="64 buckets to 1024")
    compare(dev, dt, t, do, SF.RelativeBuckets(64, 1024, False), 2, causal=True, q_start=600, what="past only")


@_dt
def test_attention_queries_that_see_nothing(dev, dt):
    """Whatever q and dout hold in rows without a key, no gradient shows it."""
    bk = SF.RelativeBuckets(16, 24, True)
    *t, do = case(32, dt, 2, 2, 1, 24, 45, 70)
    keep = torch.ones(2, 70)
    keep[1] = 0
    t[0][0, :, :9] = float("nan")                                         # (q_start = -9, causal: queries 0 .. 8 see nothing)
    t[0][1] = float("inf")
    do[0, :, 3] = float("nan")
    do[1, 0] = float("inf")
    ls = [x.to(dev).requires_grad_() for x in t]
    out = SF.bucket_attention(*ls, bk, 2, keep=keep.to(dev), causal=True, q_start=-9)
    assert not out[0, :, :9].any() and not out[1].any()
    grads = torch.autograd.grad(out, ls, do.to(dev))
    clean = [t[0].clone(), *t[1:]]
    clean[0][0, :, :9] = 1.0
    clean[0][1] = 1.0
    do = torch.nan_to_num(do.clone(), 0.0, 0.0, 0.0)
    lc = [x.to(dev).requires_grad_() for x in clean]
    want = torch.autograd.grad(SF.bucket_attention(*lc, bk, 2, keep=keep.to(dev), causal=True, q_start=-9), lc, do.to(dev))
    for g, w in zip(grads, want):
        assert torch.equal(g, w)


@_dt
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_attention_buckets_without_weight(dev, dt, low):
    """A table entry of -inf or the type's lowest value hides its bucket's pairs, as `keep` would."""
    bk = SF.RelativeBuckets(16, 24, True)
    for tq, tk in ((40, 70), (1, 130)):
        *t, do = case(33, dt, 1, 2, 2, 24, tq, tk)
        t[3][7, 0] = low                                                 # (head 0: the keys far in the past)
        t[3][8:, 1] = low                                                # (head 1: all keys behind the query)
        compare(dev, dt, t, do, bk, 2, q_start=30, what=f"{tq}")


def test_second_derivatives_are_refused(dev):
    gen = torch.Generator().manual_seed(34)
    bk = SF.RelativeBuckets(8, 20)
    x = torch.randn(1, 16, 9, generator=gen).to(dev).requires_grad_()
    table = torch.randn(8, 2, generator=gen).to(dev).requires_grad_()
    for out in (SF.layer_norm_nct(x, None, None), SF.bucket_attention(x, x, x, table, bk, 2), SF.bucket_bias(table, bk, 3, 4)):
        leaf = x if out.shape == x.shape else table
        g, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaf)


def test_far_positions_and_lengths(dev):
    """Starts beyond the ABI's 32 bits are as far as can be; lengths beyond them are refused before anything is allocated."""
    bk = SF.RelativeBuckets(8, 20)
    table = torch.randn(8, 2, generator=torch.Generator().manual_seed(35)).to(dev).requires_grad_()
    for start, bucket in ((1 << 40, 3), (-(1 << 40), 7)):
        bias = SF.bucket_bias(table, bk, 3, 5, q_start=start)
        assert torch.equal(bias, table[bucket][:, None, None].expand(2, 3, 5))
        g, = torch.autograd.grad(bias.sum(), table)
        want = torch.zeros(8, 2)
        want[bucket] = 15
        assert torch.equal(g.cpu(), want)
        q = torch.randn(1, 8, 3, generator=torch.Generator().manual_seed(36)).to(dev)
        assert torch.equal(SF.bucket_attention(q, q, q, table, bk, 2, q_start=start), SF.bucket_attention(q, q, q, table, bk, 2, q_start=99 * (1 if start > 0 else -1)))
    with pytest.raises(ValueError):
        SF.bucket_bias(table, bk, 1 << 40, 0)
    with pytest.raises(ValueError):
        SF.bucket_attention(torch.zeros(1, 2, 1, device=dev).expand(1, 2, (1 << 32) + 5)[:, :, :0], *[torch.zeros(1, 2, 0, device=dev).expand((1 << 32) + 1, 2, 0)] * 2,
                            table, bk, 2)


def test_layer_norm_nct_affine_sizes(dev):
    """gamma and beta of another size are refused with and without gradients; any stride of them is taken."""
    x = torch.randn(2, 12, 9, generator=torch.Generator().manual_seed(37)).to(dev)
    wide = torch.randn(24, generator=torch.Generator().manual_seed(38)).to(dev)
    for leaf in (x, x.clone().requires_grad_()):
        for bad in (wide, wide[:11]):
            with pytest.raises(ValueError):
                SF.layer_norm_nct(leaf, bad, None)
            with pytest.raises(ValueError):
                SF.layer_norm_nct(leaf, wide[:12], bad)
        assert torch.equal(SF.layer_norm_nct(leaf, wide[::2], wide[1::2]), SF.layer_norm_nct(leaf, wide[::2].clone(), wide[1::2].clone()))


# ---- on the GPU: real lengths, streams, graphs ----------------------------------------------------------------------------
@pytest.mark.gpu
@_dt
@pytest.mark.parametrize("shape", [(1, 4, 2, 64, 2000, 2000), (2, 2, 2, 128, 1030, 1500), (9, 8, 8, 16, 600, 513), (3, 2, 1, 96, 777, 1025)])
def test_attention_long(gpu_only, dt, shape):
    B, H, Hkv, dk, tq, tk = shape
    *t, do = case(sum(shape), dt, *shape, n=32)
    keep = torch.ones(B, tk)
    keep[0, tk - 77:] = 0
    keep[0, 300:420] = 0
    compare("cuda", dt, t, do, SF.RelativeBuckets(32, 128, True), H, keep=keep, what="masked")
    compare("cuda", dt, t, do, SF.RelativeBuckets(32, 128, False), H, causal=True, what="causal")


@pytest.mark.gpu
def test_attention_cache_beyond_32_bits(gpu_only):
    """The last entry of a cache of more than 2^32 elements: one token, several (another form), and its gradients."""
    B, H, Hkv, dk, tk = 5, 8, 8, 128, 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(41)
    k, v = (torch.randn(B, Hkv * dk, tk, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert k.numel() > 1 << 32
    table = torch.randn(32, H, generator=gen, device="cuda")
    bk = SF.RelativeBuckets(32, 128, False)
    for tq in (1, 40):
        q = torch.randn(B, H * dk, tq, generator=gen, device="cuda", dtype=torch.bfloat16)
        do = torch.randn(B, H * dk, tq, generator=gen, device="cuda", dtype=torch.bfloat16)
        ls = [x.detach().requires_grad_() for x in (q, k, v)] if tq > 1 else [q, k, v]
        out = SF.bucket_attention(*ls, table, bk, H, causal=True)
        grads = torch.autograd.grad(out, ls, do) if tq > 1 else None
        for b, h in ((0, 0), (B - 1, H - 1)):
            qh, kh, vh, dh = (x[b, h * dk:(h + 1) * dk].detach().double() for x in (q, k, v, do))
            off = torch.arange(tk, device="cuda")[None] - (tk - tq + torch.arange(tq, device="cuda")[:, None])
            lut = bucket_index(bk, 1, 400, 399)[0].to("cuda")              # offsets -399 .. 0
            s = qh.t() @ kh * dk ** -0.5 + table[:, h].double()[lut[(off.clamp(-399, 0) + 399)]]
            p = torch.softmax(s.masked_fill(off > 0, -math.inf), 1)
            near(out[b, h * dk:(h + 1) * dk], (vh @ p.t()).cpu(), 3 * UBF, f"out {tq} {b}")
            if grads:
                dp = dh.t() @ vh
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * dk ** -0.5
                near(grads[0][b, h * dk:(h + 1) * dk], (kh @ ds.t()).cpu(), 3 * UBF, f"dq {b}")
                near(grads[1][b, h * dk:(h + 1) * dk], (qh @ ds).cpu(), 3 * UBF, f"dk {b}")
                near(grads[2][b, h * dk:(h + 1) * dk], (dh @ p).cpu(), 3 * UBF, f"dv {b}")


@pytest.mark.gpu
def test_bucket_bias_many_rows(gpu_only):
    """More rows than a launch has workgroups in its second dimension."""
    tq = (1 << 20) + 3
    bk = SF.RelativeBuckets(8, 20)
    table = torch.randn(8, 1, device="cuda").requires_grad_()
    bias = SF.bucket_bias(table, bk, tq, 3, q_start=-10)
    g, = torch.autograd.grad(bias, table, torch.ones_like(bias))
    want = torch.zeros(8)
    for o in range(-60, 40):
        rows = sum(1 for j in range(3) if 0 <= j - o + 10 < tq)
        want[bucket_of(o, 8, 20, True)] += rows
    far = 3 * tq - int(want.sum())
    want[bucket_of(-1000, 8, 20, True)] += far
    assert torch.equal(g[:, 0].cpu(), want)                               # (whole numbers below 2^24)


def _block(x, gamma, beta, table, bk, H):
    n = SF.layer_norm_nct(x, gamma, beta)
    return SF.bucket_attention(n, n, n, table, bk, H, causal=True)


@pytest.mark.gpu
@_dt
def test_block_on_another_stream(gpu_only, dt):
    """Forward and backward on a side stream that made the inputs: the same bits as on the default stream."""
    gen = torch.Generator().manual_seed(42)
    raw = [torch.randn(3, 64, 500, generator=gen).to(DT[dt]), torch.rand(64, generator=gen), torch.randn(64, generator=gen), torch.randn(16, 2, generator=gen),
           torch.randn(3, 64, 500, generator=gen).to(DT[dt])]
    bk = SF.RelativeBuckets(16, 40, False)

    def run():
        *ls, do = [x.cuda() for x in raw]
        ls = [x.requires_grad_() for x in ls]
        out = _block(*ls, bk, 2)
        return [out, *torch.autograd.grad(out, ls, do)]
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def _replays(graphs, inputs, outputs, fresh, eager):
    """Replays the graphs in turn over new inputs, eager work and a synchronization between them, against the eager result."""
    for _ in range(4):
        for src, dst in zip(fresh(), inputs):
            dst.copy_(src)
        want = eager()
        torch.cuda.synchronize()
        for g, out in zip(graphs, outputs):
            g.replay()
            torch.cuda.synchronize()
            for a, w in zip(out, want):
                assert torch.equal(a, w)
            eager()


@pytest.mark.gpu
@_dt
def test_cached_token_in_graphs(gpu_only, dt):
    """The serving form captured twice (the splits' workspaces are each graph's own), with moving lengths."""
    gen = torch.Generator(device="cuda").manual_seed(43)
    B, H, Hkv, dk, tk = 3, 8, 2, 40, 2000
    bk = SF.RelativeBuckets(32, 128, False)
    shapes = ((B, H * dk, 1), (B, Hkv * dk, tk), (B, Hkv * dk, tk))
    table = torch.randn(32, H, device="cuda", generator=gen)

    def fresh():
        return [torch.randn(s, device="cuda", generator=gen).to(DT[dt]) for s in shapes] + [torch.randint(0, tk, (B,), device="cuda", generator=gen).int()]
    inputs = fresh()

    def eager():
        with torch.no_grad():
            return [SF.bucket_attention(*inputs[:3], table, bk, H, causal=True, q_start=inputs[3])]
    eager()
    graphs, outputs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs.append(eager())
        graphs.append(g)
    _replays(graphs, inputs, outputs, fresh, eager)


@pytest.mark.gpu
@_dt
def test_block_training_step_in_a_graph(gpu_only, dt):
    """Norm and attention with all gradients captured; leaves of their own in the graph."""
    gen = torch.Generator(device="cuda").manual_seed(44)
    bk = SF.RelativeBuckets(16, 40, False)

    def fresh():
        return [torch.randn(2, 96, 300, device="cuda", generator=gen).to(DT[dt]), torch.rand(96, device="cuda", generator=gen),
                torch.randn(96, device="cuda", generator=gen), torch.randn(16, 2, device="cuda", generator=gen),
                torch.randn(2, 96, 300, device="cuda", generator=gen).to(DT[dt])]
    inputs = fresh()

    def step():
        ls = [x.detach().requires_grad_() for x in inputs[:4]]
        out = _block(*ls, bk, 2)
        return [out.detach(), *torch.autograd.grad(out, ls, inputs[4])]
    step()
    graphs, outputs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs.append(step())
        graphs.append(g)
    _replays(graphs, inputs, outputs, fresh, step)
