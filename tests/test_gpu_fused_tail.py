"""GPU tests of the attention and dense-layer kernels (vx_attn.hip, vx_linear.hip, vista_amd/fused_tail.py) against plain
float64 evaluations of the same formulas.

Tolerances are elementwise bounds worked out from the arithmetic, not fitted. u = 2^-24.
  product     sum_k a_k b_k over K terms in fp32 accumulators. fp32 operands: three planes, h the top 16 bits of x, so
              |m| < 2^-7 |x| and |l| < 2^-15 |x|; the dropped products m l, l m, l l are below 2^-21 |a||b|. 6 ceil(K/32) matrix
              instructions (one for bf16) each add once to the accumulator and add up 32 products inside (5 levels), every
              addition off by at most 2^-23 of the running magnitude. Error <= gamma(K) sum |a||b|,
              gamma = [2^-21 +] 2^-23 (n + 5 n / ceil(K/32)), n = instructions of one element; a sum cut into slabs adds one
              addition a slab, covered by 2^-23 * 64.
  output      rounded once: finfo.eps / 2 of the value.
  attention   a score is off by ds = scale gamma(D) sum |q||k| + 2^-22 |s|; p = exp(s - m) / l is off by 2 max ds + 2^-20
              relative (statistics, exp2 and the division), for bf16 by another 2^-8 where it is a matrix operand; the rest
              is products. Gradients carry these through their formulas, with |.| in the place of every factor.
"""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def gamma(k, dtype):
    steps = max(1, -(-k // 32))
    n = steps * (6 if dtype == F32 else 1)
    return (2.0 ** -21 if dtype == F32 else 0.0) + 2.0 ** -23 * (n + 5 * n / steps + 64)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, bound, what):
    d = (got.double() - want).abs()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    worst = (d / (bound + 1e-300)).max().item() if d.numel() else 0.0
    assert worst <= 1.0, (what, worst, d.max().item())


# ------------------------------------------------------------------------------------------------ dense layer
def act64(a, act):
    f = torch.nn.functional
    return {"none": lambda t: t, "relu": torch.relu, "gelu": f.gelu, "silu": f.silu}[act](a)


def slope64(a, act):
    if act == "none":
        return torch.ones_like(a)
    if act == "relu":
        return (a > 0).double()
    if act == "gelu":
        return torch.special.ndtr(a) + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(a)
    return s * (1 + a * (1 - s))


def make_linear(m, k, n, dtype, dev, seed, bias, residual):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    return (r(m, k).to(dtype), (r(n, k) * k ** -0.5).to(dtype), (r(n) * 0.3).to(dtype) if bias else None,
            r(m, n).to(dtype) if residual else None, r(m, n).to(dtype))


LINEAR = [(1, 1, 1), (1, 384, 512), (7, 384, 512), (63, 33, 65), (64, 64, 64), (65, 31, 129), (130, 7, 3), (257, 100, 255),
          (1600, 384, 384), (999, 511, 77), (16385, 64, 300), (20000, 72, 130)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act,bias,residual", [("none", False, False), ("none", True, True), ("relu", True, False),
                                               ("relu", True, True), ("gelu", True, True), ("silu", False, True)])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_forward(m, k, n, act, bias, residual, dtype, dev):
    from vista_amd import ops
    x, w, b, r, _ = make_linear(m, k, n, dtype, dev, m + 7 * k + n, bias, residual)
    y, pre = ops.linear_fwd(x, w, b, r, act, want_pre=True)
    a = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()
    for t in (b, r):
        if t is not None:
            a, size = a + t.double(), size + t.double().abs()
    off = gamma(k, dtype) * size
    within(pre, a, off + half_step(dtype) * (a.abs() + off) + 1e-38, "pre")
    want = act64(a, act)
    # slopes of all four are at most 1.13; the activation itself is good to 2^-21 of its argument
    off = 1.13 * off + 2.0 ** -21 * a.abs()
    within(y, want, off + half_step(dtype) * (want.abs() + off) + 1e-38, "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_backward(m, k, n, act, dtype, dev):
    from vista_amd import ops
    x, w, _, s, dy = make_linear(m, k, n, dtype, dev, 3 * m + k + n, False, True)
    saved = {"none": None, "relu": s.clamp(min=0)}.get(act, s)
    dx, dw, db, dpre = ops.linear_bwd(dy, x, w, act, saved)
    g = dy.double() * (slope64(s.double(), act) if act != "none" else 1.0)
    # the slope is good to 2^-20 (exp and erf of a few), g is rounded to the tensors' type
    goff = (2.0 ** -20 if act in ("gelu", "silu") else 0.0) * dy.double().abs() * (1 + s.double().abs())
    goff = goff + (half_step(dtype) * g.abs() if act in ("gelu", "silu") else 0.0)
    within(dpre, g, goff + 1e-38, "dpre")
    wd, xd = w.double().abs(), x.double().abs()
    want = g @ w.double()
    off = gamma(n, dtype) * (g.abs() @ wd) + goff @ wd
    within(dx, want, off + half_step(dtype) * (want.abs() + off) + 1e-38, "dx")
    want = g.t() @ x.double()
    off = gamma(m, dtype) * (g.abs().t() @ xd) + goff.t() @ xd
    within(dw, want, off + half_step(dtype) * (want.abs() + off) + 1e-38, "dw")
    want = g.sum(0)
    # a thread's column sum runs over at most m / 8 rows one after the other, then over lanes and chunks
    off = 2.0 ** -24 * (min(m, 8192) / 8 + 1100) * g.abs().sum(0) + goff.sum(0)
    within(db, want, off + half_step(dtype) * (want.abs() + off) + 1e-38, "dbias")


def test_linear_reads_strides_in_place(dev):
    from vista_amd import ops
    g = torch.Generator(device=dev).manual_seed(4)
    wide = torch.randn((300, 2, 96), generator=g, device=dev)
    big_w = torch.randn((70, 200), generator=g, device=dev)
    row = torch.randn((1, 70), generator=g, device=dev)
    x, w, r = wide[:, 1], big_w[:, 3:99], row.expand(300, 70)          # row strides 192, 200 and 0, bases off 16 bytes
    want, _ = ops.linear_fwd(x.contiguous(), w.contiguous(), None, r.contiguous())
    assert torch.equal(ops.linear_fwd(x, w, None, r)[0], want)
    assert torch.equal(ops.linear_fwd(x.t().contiguous().t(), w, None, r)[0], want)       # last dimension strided: copied
    dy = torch.randn((300, 140), generator=g, device=dev)[:, 1::2]
    one, two = ops.linear_bwd(dy, x, w), ops.linear_bwd(dy.contiguous(), x.contiguous(), w.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [1, 3, 31, 33, 1000, 6401])
def test_linear_gradients_read_no_row_behind_the_last(m, dtype, dev):
    """Operands at the front of a buffer whose other rows are NaN."""
    from vista_amd import ops
    x, w, _, s, dy = make_linear(m, 384, 512, dtype, dev, m, False, True)
    want = ops.linear_bwd(dy, x, w, "relu", s)

    def front(t):
        buf = torch.full((m + 70, t.shape[1]), math.nan, dtype=dtype, device=dev)
        buf[:m] = t
        return buf[:m]

    for a, b in zip(ops.linear_bwd(front(dy), front(x), w, "relu", front(s)), want):
        assert torch.equal(a, b)
    assert torch.equal(ops.linear_fwd(front(x), w)[0], ops.linear_fwd(x, w)[0])
    one = ops.linear_bwd(dy, x[:1].expand(m, 384), w, "none")            # a repeated row: stride 0
    for a, b in zip(one, ops.linear_bwd(dy, x[:1].expand(m, 384).contiguous(), w, "none")):
        within(a, b.double(), 2 * gamma(max(m, 512), dtype) * 64 * (1 + b.double().abs()) + 4 * half_step(dtype) * b.double().abs(), "row")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 70, 50, 4, 2, 2, 24, 40), (1, 300, 100, 2, 2, 1, 192, 384), (1, 300, 45, 2, 2, 1, 160, 200)])
def test_attention_reads_no_row_behind_the_last(shape, dtype, dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, 2, "some")
    want, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    grads = ops.attn_bwd(do, q, k, v, want, stats, km)
    free, fstats = ops.attn_fwd(q, k, v, want_stats=True)
    fgrads = ops.attn_bwd(do, q, k, v, free, fstats)

    def front(t):
        buf = torch.full((t.shape[0], t.shape[1] + 130, *t.shape[2:]), math.nan, dtype=dtype, device=dev)
        buf[:, :t.shape[1]] = t
        return buf[:, :t.shape[1]]

    q2, k2, v2, do2 = (front(t) for t in (q, k, v, do))
    for mask, first, back in ((km, want, grads), (None, free, fgrads)):
        out, st = ops.attn_fwd(q2, k2, v2, mask, want_stats=True)
        assert torch.equal(out, first)
        assert all(torch.equal(a, b) for a, b in zip(ops.attn_bwd(do2, q2, k2, v2, out, st, mask), back))


def test_linear_without_rows(dev):
    from vista_amd import ops
    w = torch.randn(5, 9, device=dev)
    y, _ = ops.linear_fwd(torch.empty(0, 9, device=dev), w)
    assert y.shape == (0, 5)
    dx, dw, db, _ = ops.linear_bwd(torch.empty(0, 5, device=dev), torch.empty(0, 9, device=dev), w)
    assert dx.shape == (0, 9) and not dw.any() and not db.any() and dw.shape == (5, 9)


def test_linear_nan_and_inf_stay_in_their_row(dev):
    from vista_amd import ops
    x, w, b, _, _ = make_linear(130, 64, 96, F32, dev, 1, True, False)
    clean, _ = ops.linear_fwd(x, w, b, act="relu")
    x[17, 3], x[99, 0] = math.nan, math.inf
    y, _ = ops.linear_fwd(x, w, b, act="relu")
    keep = torch.ones(130, dtype=torch.bool, device=dev)
    keep[17] = keep[99] = False
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[17]).all()


def off_by_its_rounding(got, want, what, room):
    """A bf16 result whose value before the rounding is good to 2^-15: the 2-norm of its error is that of the rounding alone, r (rms some
    2^-9 / sqrt 3 of each value), times sqrt(1 + (2^-15 / r)^2) < 1.001; `room` for the values that the rounding itself leaves exact."""
    rounding = (want.to(BF16).double() - want).norm()
    assert (got.double() - want).norm() <= room * rounding, (what, ((got.double() - want).norm() / rounding).item())


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(50, 70, 90), (3000, 128, 96), (20000, 128, 256)])
def test_bf16_layer_gradients_are_rounded_once(m, k, n, act, dev):
    """dx and dw of a smooth activation: g = dy act'(pre) goes into both products unrounded."""
    from vista_amd import ops
    x, w, _, s, dy = make_linear(m, k, n, BF16, dev, m, False, True)
    dx, dw, db, dpre = ops.linear_bwd(dy, x, w, act, s)
    g = dy.double() * slope64(s.double(), act)
    for name, got, want in (("dpre", dpre, g), ("dx", dx, g @ w.double()), ("dw", dw, g.t() @ x.double()), ("dbias", db, g.sum(0))):
        off_by_its_rounding(got, want, name, 1.02)


# ------------------------------------------------------------------------------------------------ attention
# batch, q_len, k_len, heads, k_heads, v_heads, dim, v_dim
ATTN = [(1, 1, 1, 1, 1, 1, 1, 1), (1, 1, 480, 2, 2, 1, 192, 384), (2, 65, 33, 4, 2, 1, 37, 53), (1, 130, 100, 2, 2, 1, 24, 48),
        (2, 77, 129, 3, 1, 3, 96, 192), (1, 200, 65, 2, 2, 2, 128, 128), (3, 17, 64, 6, 3, 2, 64, 64), (2, 40, 31, 2, 1, 2, 33, 100),
        (1, 64, 32, 1, 1, 1, 32, 64), (2, 150, 300, 2, 2, 1, 192, 384), (1, 3, 5000, 2, 1, 1, 48, 48), (5, 1, 7, 3, 3, 1, 130, 257)]
# enough query tiles for the 128-query form, in the smallest and the largest tile
ATTN_WIDE = [(2, 2048, 70, 8, 8, 8, 16, 24), (4, 4096, 40, 2, 2, 1, 192, 384), (2, 2050, 65, 8, 2, 4, 96, 130)]
# five and more tiles of 64 queries, every width class, lists of keys longer than one sweep
ATTN_IMAGES = [(1, 300, 100, 2, 2, 1, 192, 384), (2, 333, 77, 4, 2, 1, 37, 53), (1, 321, 130, 2, 1, 2, 24, 48), (1, 400, 65, 1, 1, 1, 64, 64),
               (2, 270, 200, 2, 2, 1, 128, 128), (1, 300, 260, 2, 2, 2, 90, 180), (1, 260, 33, 2, 2, 1, 60, 100),
               (2, 300, 3001, 2, 1, 1, 48, 48), (1, 257, 1, 1, 1, 1, 8, 8), (1, 290, 70, 2, 2, 1, 136, 264),
               (1, 5000, 3, 2, 1, 1, 16, 16)]
MASKS = ["none", "some", "blank", "all"]


def make_attn(shape, dtype, dev, seed, mask, poison=False):
    b, sq, sk, h, hk, hv, d, dv = shape
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=dev).to(dtype)  # noqa: E731
    q, k, v, do = r(b, sq, h, d), r(b, sk, hk, d), r(b, sk, hv, dv), r(b, sq, h, dv)
    km = None
    if mask != "none":
        km = torch.rand((b, sk), generator=g, device=dev) > 0.4
        if mask == "blank":
            km[0] = False
        elif mask == "all":
            km[:] = False
        if poison:                      # what masked rows hold must not matter
            bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], device=dev, dtype=dtype)
            where = ~km
            k[where] = bad[torch.randint(4, (int(where.sum()), hk, d), generator=g, device=dev)]
            v[where] = bad[torch.randint(4, (int(where.sum()), hv, dv), generator=g, device=dev)]
    return q, k, v, km, do


def attn_reference(q, k, v, km, do, scale=None):
    """float64 values and elementwise bounds of out, dq, dk, dv."""
    dt = q.dtype
    b, sq, h, d = q.shape
    sk, hk, hv, dv = k.shape[1], k.shape[2], v.shape[2], v.shape[3]
    scale = d ** -0.5 if scale is None else scale
    gk, gv = h // hk, h // hv
    live = torch.ones((b, sk), dtype=torch.bool, device=q.device) if km is None else km
    z = lambda t: t.double().masked_fill(~live[:, :, None, None], 0.0)  # noqa: E731
    Q, G = q.double().transpose(1, 2), do.double().transpose(1, 2)
    K, V = z(k).transpose(1, 2).repeat_interleave(gk, 1), z(v).transpose(1, 2).repeat_interleave(gv, 1)
    L = live[:, None, None, :]
    s = (scale * (Q @ K.transpose(2, 3))).masked_fill(~L, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e300) if sk else s.new_zeros((b, h, sq, 1))
    p = torch.exp(s - m)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = p @ V
    ds_ = abs(scale) * gamma(d, dt) * (Q.abs() @ K.abs().transpose(2, 3)) + 2.0 ** -22 * s.masked_fill(~L, 0.0).abs()
    ds_ = ds_.masked_fill(~L, 0.0)
    rel = 2 * (ds_.amax(-1, keepdim=True) if sk else s.new_zeros((b, h, sq, 1))) + 2.0 ** -20
    r16 = 2.0 ** -8 if dt == BF16 else 0.0
    hs = half_step(dt)
    done = lambda val, off: off + hs * (val.abs() + off) + 1e-38  # noqa: E731
    pv = p @ V.abs()
    b_out = done(out, (rel * 1.01 + r16 + gamma(sk, dt)) * pv)
    dV = p.transpose(2, 3) @ G
    b_dV = (p * (rel * 1.01 + r16 + gamma(sq, dt))).transpose(2, 3) @ G.abs()
    dP = G @ V.transpose(2, 3)
    delta = (G * out).sum(-1, keepdim=True)
    dS = scale * p * (dP - delta)
    b_dP = gamma(dv, dt) * (G.abs() @ V.abs().transpose(2, 3))
    b_delta = (G.abs() * b_out).sum(-1, keepdim=True) + 2.0 ** -24 * 16 * (G.abs() * out.abs()).sum(-1, keepdim=True)
    e_dS = abs(scale) * p * ((rel * 1.01 + 2.0 ** -22) * (dP - delta).abs() + b_dP + b_delta)
    e_dS = e_dS + r16 * (dS.abs() + e_dS)
    dQ, dK = dS @ K, dS.transpose(2, 3) @ Q
    b_dQ = e_dS @ K.abs() + gamma(sk, dt) * (dS.abs() @ K.abs())
    b_dK = e_dS.transpose(2, 3) @ Q.abs() + gamma(sq, dt) * (dS.abs().transpose(2, 3) @ Q.abs())
    fold = lambda t, g: t.view(b, h // g, g, *t.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
    dK, b_dK, dV, b_dV = fold(dK, gk), fold(b_dK, gk), fold(dV, gv), fold(b_dV, gv)
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    return {"out": (t(out), t(b_out)), "dq": (t(dQ), done(t(dQ), t(b_dQ))), "dk": (dK, done(dK, b_dK)), "dv": (dV, done(dV, b_dV))}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("shape", ATTN + ATTN_IMAGES)
def test_attention_and_gradients(shape, mask, dtype, dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, sum(shape), mask, poison=True)
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    dq, dk, dv = ops.attn_bwd(do, q, k, v, out, stats, km)
    within(dq, *ref["dq"], "dq")
    within(dk, *ref["dk"], "dk")
    within(dv, *ref["dv"], "dv")
    if km is not None:
        assert not dk[~km].any() and not dv[~km].any()
        assert not out[~km.any(1)].any() and not dq[~km.any(1)].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", ATTN_WIDE)
def test_attention_many_queries(shape, dtype, dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, 5, "blank", poison=True)
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


def stale(*sizes, dev):
    """Leaves NaN in the memory that the next tensors of these sizes get: a row that a kernel does not write shows."""
    held = [torch.full((n,), math.nan, dtype=F32, device=dev) for n in sizes for _ in range(4)]
    del held


# batch x heads x query tiles enough for the 128-query form, but few queries of each
ATTN_MANY_SHORT = [(64, 100, 20, 8, 8, 8, 64, 64), (16, 512, 33, 8, 8, 8, 48, 48), (128, 128, 20, 2, 2, 1, 192, 384),
                   (6, 500, 40, 6, 6, 6, 150, 300), (90, 65, 17, 8, 4, 2, 24, 30), (70, 257, 21, 8, 8, 8, 33, 65), (130, 256, 9, 4, 4, 4, 96, 128),
                   (128, 320, 30, 2, 2, 1, 190, 380)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", ["none", "blank"])
@pytest.mark.parametrize("shape", ATTN_MANY_SHORT)
def test_attention_of_many_short_sequences_writes_every_row(shape, mask, dtype, dev):
    """Many heads of 65 to 512 queries each: every row of out and stats is written, whatever tile the launch takes."""
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, sum(shape), mask, poison=True)
    ref = attn_reference(q, k, v, km, do)
    stale(ref["out"][0].numel() * q.element_size() // 4, shape[0] * shape[3] * shape[1] * 2, dev=dev)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    assert not torch.isnan(stats).any()
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k_len", [1023, 1025, 2047, 2048, 2049])
def test_attention_around_the_longest_short_mask(k_len, dtype, dev):
    """Lists of 1024 keys a sweep; masks of at most 2048 keys are listed by the workgroups that use them."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 270, k_len, 2, 2, 1, 40, 72), dtype, dev, k_len, "some", poison=True)
    km[0, :], km[0, -1] = False, True                   # the last key alone
    k[0, -1], v[0, -1] = 0.5, 0.25
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


@pytest.mark.parametrize("k_len", [2000, 5001])
def test_attention_gradients_in_chunks_of_queries(k_len, dev):
    """Many queries: one chunk of several splits (2000 keys), and more probabilities than the workspace holds at once (5001)."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((1, 20000, k_len, 2, 2, 1, 16, 24), F32, dev, 6, "some", poison=True)
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


@pytest.mark.parametrize("scale", [None, 1.0])
@pytest.mark.parametrize("shape", [(1, 3, 700, 2, 2, 1, 64, 96), (2, 200, 150, 2, 2, 1, 48, 48), (2, 700, 300, 4, 2, 1, 96, 192),
                                   (1, 600, 900, 2, 2, 1, 192, 384), (8, 1100, 140, 8, 8, 8, 64, 64)])
def test_bf16_attention_is_rounded_once(shape, scale, dev):
    """Every width of tile, few and many queries, split and joined keys; flat and peaked (scale 1) rows."""
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, BF16, dev, 21, "some")
    ref = attn_reference(q, k, v, km, do, scale)
    off_by_its_rounding(ops.attn_fwd(q, k, v, km, scale)[0], ref["out"][0], "out", 1.02)


@pytest.mark.parametrize("scale", [None, 1.0])
@pytest.mark.parametrize("shape", [(1, 100, 200, 2, 2, 1, 64, 96), (3, 777, 301, 4, 2, 1, 96, 192), (1, 3000, 500, 2, 2, 1, 192, 384),
                                   (4, 2000, 260, 4, 4, 4, 64, 64), (1, 700, 1000, 2, 2, 1, 144, 168)])
def test_bf16_attention_gradients_are_rounded_once(shape, scale, dev):
    """More than 128 keys, every tile of the backward pass, flat rows and (scale 1) rows that few keys dominate."""
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, BF16, dev, 22, "some")
    ref = attn_reference(q, k, v, km, do, scale)
    out, stats = ops.attn_fwd(q, k, v, km, scale, want_stats=True)
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km, scale)):
        off_by_its_rounding(got, ref[name][0], name, 1.02)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_gradients_over_many_chunks(dtype, dev):
    """Few queries over very many keys: four chunks of equal length whose last is shorter; dk and dv are summed over all of them."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((1, 3100, 60001, 1, 1, 1, 16, 24), dtype, dev, 16, "some", poison=True)
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    stale(1 << 28, dev=dev)
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


def test_attention_gradients_of_very_many_rows(dev):
    """More rows than the waves of one launch that sums dout * out: 64 x 16 x 4200 of them. The first and the last batch by themselves."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((64, 4200, 130, 16, 1, 1, 8, 8), BF16, dev, 17, "some")
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    grads = ops.attn_bwd(do, q, k, v, out, stats, km)
    for b in (slice(0, 1), slice(63, 64)):
        ref = attn_reference(q[b], k[b], v[b], km[b], do[b])
        for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            within(got[b], *ref[name], name)


@pytest.mark.parametrize("k_len,live", [(2, 2), (5, 3), (16, 10), (40, 26), (128, 128)])
def test_bf16_gradients_over_few_keys_lose_nothing(k_len, live, dev):
    """Over at most 128 keys P and dS are 16-bit operands and delta is summed from P dP itself: what is left beside the gradients' own
    rounding to bf16 (2-norm, rms about 2^-9 of each value) is 2^-17 of the operands: 1.05 of it with room for the sample."""
    from vista_amd import ops
    q, k, v, _, do = make_attn((1, 600, k_len, 2, 2, 1, 64, 96), BF16, dev, k_len, "none")
    km = (torch.arange(k_len, device=dev) < live)[None]
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    ref = attn_reference(q, k, v, km, do)
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        want = ref[name][0]
        rounding = (want.to(BF16).double() - want).norm()
        assert (got.double() - want).norm() <= 1.05 * rounding, name


def test_attention_of_large_scores(dev):
    """Scores of some hundreds: the running maximum keeps every exponent in range; scale 0 and below zero are scales too."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 70, 90, 2, 2, 1, 64, 64), F32, dev, 9, "some")
    for scale in (40.0, -3.0, 0.0):
        ref = attn_reference(q, k, v, km, do, scale)
        out, stats = ops.attn_fwd(q, k, v, km, scale, want_stats=True)
        within(out, *ref["out"], "out")
        for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km, scale)):
            within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 5, 40, 2, 2, 1, 32, 48), (1, 3, 3000, 1, 1, 1, 64, 64), (2, 300, 200, 2, 2, 1, 48, 96)])
def test_scores_past_the_range_are_no_missing_keys(shape, dtype, dev):
    """A query whose scores all overflow (to -inf, or to +inf when scaled) has keys: NaN, not the zeros of a query without any; the
    other queries do not see it. Direct, split and packed keys."""
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, 31, "some")
    km[:, -1] = True
    k[..., 0] = k[..., 0].abs() + 0.5
    q[:, 1] = 0.0
    q[:, 1, :, 0] = -1e38                                  # scores of -1e37 and below, all of one sign
    kk = k * 100.0                                         # ... past -3.4e38: -inf
    rest = torch.ones(shape[1], dtype=torch.bool, device=dev)
    rest[1] = False
    out, st = ops.attn_fwd(q, kk, v, km, 0.01 * shape[6] ** -0.5, want_stats=True)
    assert torch.isnan(out[:, 1]).all() and torch.isfinite(out[:, rest]).all()
    dq, dk, dv = ops.attn_bwd(do, q, kk, v, out, st, km, 0.01 * shape[6] ** -0.5)
    assert torch.isnan(dq[:, 1]).all() and torch.isfinite(dq[:, rest]).all()
    q[:, 1, :, 0] = 1e37                                   # finite scores, above the range when scaled
    k[..., 0] = 2.0
    out, st = ops.attn_fwd(q, k, v, km, 1e3, want_stats=True)
    assert torch.isnan(out[:, 1]).all() and torch.isfinite(out[:, rest]).all()
    km[0] = False                                          # without keys: zeros all the same
    out, st = ops.attn_fwd(q, k, v, km, 1e3, want_stats=True)
    assert not out[0].any() and not ops.attn_bwd(do, q, k, v, out, st, km, 1e3)[0][0].any()


def test_attention_without_keys_or_queries(dev):
    from vista_amd import ops
    q, k, v = (torch.randn(2, n, 2, 16, device=dev) for n in (5, 0, 0))
    out, stats = ops.attn_fwd(q, k, v, want_stats=True)
    assert out.shape == (2, 5, 2, 16) and not out.any()
    dq, dk, dv = ops.attn_bwd(torch.ones_like(out), q, k, v, out, stats)
    assert not dq.any() and dk.shape == k.shape and dv.shape == v.shape
    q, k, v = (torch.randn(2, n, 2, 16, device=dev) for n in (0, 5, 5))
    out, stats = ops.attn_fwd(q, k, v, want_stats=True)
    assert out.shape == (2, 0, 2, 16)
    dq, dk, dv = ops.attn_bwd(out, q, k, v, out, stats)
    assert dq.shape == q.shape and not dk.any() and not dv.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_reads_strides_in_place(dtype, dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 70, 50, 4, 2, 2, 24, 40), dtype, dev, 2, "some")
    want, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    grads = ops.attn_bwd(do, q, k, v, want, stats, km)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    kv = torch.cat([torch.zeros_like(k[..., :1]), k, v], -1)[..., 1:]             # one buffer, rows off 16 bytes
    mask_rows = torch.stack([~km, km], 1)[:, 1]
    q2, k2, v2, do2 = heads_first(q), kv[..., :24], kv[..., 24:], heads_first(do)
    out, st = ops.attn_fwd(q2, k2, v2, mask_rows, want_stats=True)
    assert torch.equal(out, want) and torch.equal(st, stats)
    for a, b in zip(ops.attn_bwd(do2, q2, k2, v2, out, st, mask_rows), grads):
        assert torch.equal(a, b)
    one = torch.ones((1, 1, 1, 1), dtype=dtype, device=dev).expand_as(do)         # a sum's gradient: all strides 0
    for a, b in zip(ops.attn_bwd(one, q, k, v, want, stats, km), ops.attn_bwd(one.contiguous(), q, k, v, want, stats, km)):
        assert torch.equal(a, b)


def test_attention_offsets_past_32_bits(dev):
    """Two batches of keys and values whose elements lie more than 2^31 apart."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 40, 50, 2, 2, 1, 32, 48), BF16, dev, 3, "some")
    far = (1 << 31) + 64
    buf = torch.empty(far + 50 * 2 * 32 + 50 * 48, dtype=BF16, device=dev)
    k2 = buf.as_strided((2, 50, 2, 32), (far, 64, 32, 1))
    v2 = buf.as_strided((2, 50, 1, 48), (far, 48, 48, 1), storage_offset=50 * 64)
    k2.copy_(k)
    v2.copy_(v)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    out2, stats2 = ops.attn_fwd(q, k2, v2, km, want_stats=True)
    assert torch.equal(out, out2)
    for a, b in zip(ops.attn_bwd(do, q, k, v, out, stats, km), ops.attn_bwd(do, q, k2, v2, out2, stats2, km)):
        assert torch.equal(a, b)


def test_same_inputs_same_bits(dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 300, 200, 2, 2, 1, 192, 384), F32, dev, 8, "some")
    runs = []
    for _ in range(3):
        out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
        runs.append((out, *ops.attn_bwd(do, q, k, v, out, stats, km)))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    x, w, _, s, dy = make_linear(5000, 130, 70, F32, dev, 1, False, True)
    a, b = ops.linear_bwd(dy, x, w, "gelu", s), ops.linear_bwd(dy, x, w, "gelu", s)
    assert all(torch.equal(i, j) for i, j in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 3, (1 << 21) + 9, 1, 1, 1, 8, 8), (70000, 2, 5, 2, 1, 2, 4, 6), (1, 2000, 2, 64, 16, 4, 8, 12)])
def test_attention_of_extreme_shapes(shape, dtype, dev):
    """Rows of scores longer than the fast loads' strides, more batches than 16 bits, many heads that share keys."""
    from vista_amd import ops
    q, k, v, km, do = make_attn(shape, dtype, dev, 41, "some", poison=True)
    ref = attn_reference(q, k, v, km, do)
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    within(out, *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), ops.attn_bwd(do, q, k, v, out, stats, km)):
        within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(5, 1 << 20, 9), (9, 8, 1 << 20), (300, 70000, 70)])
def test_linear_of_extreme_shapes(m, k, n, dtype, dev):
    from vista_amd import ops
    x, w, b, r, dy = make_linear(m, k, n, dtype, dev, 42, True, True)
    a = x.double() @ w.double().t() + b.double() + r.double()
    size = x.double().abs() @ w.double().abs().t() + b.double().abs() + r.double().abs()
    off = gamma(k, dtype) * size
    within(ops.linear_fwd(x, w, b, r)[0], a, off + half_step(dtype) * (a.abs() + off), "y")
    dx, dw, db, _ = ops.linear_bwd(dy, x, w)
    for name, got, want, off in (("dx", dx, dy.double() @ w.double(), gamma(n, dtype) * (dy.double().abs() @ w.double().abs())),
                                 ("dw", dw, dy.double().t() @ x.double(), gamma(m, dtype) * (dy.double().abs().t() @ x.double().abs())),
                                 ("db", db, dy.double().sum(0), 2.0 ** -20 * dy.double().abs().sum(0))):
        within(got, want, off + half_step(dtype) * (want.abs() + off) + 1e-38, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_c_entries_without_the_rest(dtype, dev):
    """vx_attn_fwd and vx_attn_bwd as they were: statistics of two floats a row, no rest; a workspace of the stated size and no more."""
    import ctypes
    from vista_amd import _lib, ops
    lib, code = _lib.lib(), 0 if dtype == F32 else 1
    shape = (2, 300, 170, 4, 2, 1, 40, 60)
    q, k, v, km, do = make_attn(shape, dtype, dev, 44, "some")
    want, wstats = ops.attn_fwd(q, k, v, km, want_stats=True)
    ref = attn_reference(q, k, v, km, do)
    i64 = lambda *s: (ctypes.c_int64 * len(s))(*s)  # noqa: E731
    strides = i64(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], km.stride(0))
    room = lambda n: torch.full((n + 256,), 255, dtype=torch.uint8, device=dev)  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    out, stats = torch.empty_like(want), torch.full((8 * 300 * 2 + 64,), 7.0, device=dev)
    n = lib.vx_attn_fwd_workspace_bytes(i64(*shape), code)
    ws = room(n)
    assert lib.vx_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), km.data_ptr(), i64(*shape), strides, 40 ** -0.5, out.data_ptr(),
                           stats.data_ptr(), code, ws.data_ptr(), n, stream) == 0
    assert torch.equal(out, want) and torch.equal(stats[:4800], wstats.flatten()[:4800])
    assert (stats[4800:] == 7.0).all() and (ws[n:] == 255).all()
    grads = [torch.empty_like(t) for t in (q, k, v)]
    n = lib.vx_attn_bwd_workspace_bytes(i64(*shape), code)
    ws = room(n)
    assert lib.vx_attn_bwd(do.data_ptr(), i64(*do.stride()[:3]), q.data_ptr(), k.data_ptr(), v.data_ptr(), km.data_ptr(), i64(*shape), strides,
                           out.data_ptr(), stats.data_ptr(), 40 ** -0.5, *(g.data_ptr() for g in grads), code, ws.data_ptr(), n, stream) == 0
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, *ref[name], name)
    assert (ws[n:] == 255).all()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_gradients_stay_in_their_workspace(dtype, act, dev):
    from vista_amd import _lib, ops
    lib, code = _lib.lib(), 0 if dtype == F32 else 1
    m, k, n = 1001, 70, 90
    x, w, _, s, dy = make_linear(m, k, n, dtype, dev, 45, False, True)
    want = ops.linear_bwd(dy, x, w, act, s)
    size = lib.vx_linear_bwd_act_workspace_bytes(m, n, k, _lib.VX_ACT[act], code)
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device=dev)
    dx, dw, db, dpre = (torch.empty_like(t) for t in (x, w, want[2], dy))
    assert lib.vx_linear_bwd(dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, s.data_ptr(), m, n, k, _lib.VX_ACT[act], dpre.data_ptr(),
                             dx.data_ptr(), dw.data_ptr(), db.data_ptr(), code, ws.data_ptr(), size,
                             torch.cuda.current_stream().cuda_stream) == 0
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), want)) and (ws[size:] == 255).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_inputs(dtype, dev):
    """One query for all batches, one key head and one value row for all: strides 0, and gradients summed over them by autograd."""
    from vista_amd.fused_tail import attention
    q, k, v, km, do = make_attn((3, 70, 150, 4, 2, 2, 24, 40), dtype, dev, 43, "some")
    q1, k1, v1 = q[:1].clone(), k[:, :, :1].clone(), v[:, :1].clone()
    views = lambda a, b, c: (a.expand_as(q), b.expand_as(k), c.expand_as(v))  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (q1, k1, v1)]
    whole = [t.detach().contiguous().requires_grad_(True) for t in views(*leaves)]
    one, two = attention(*views(*leaves), key_mask=km), attention(*whole, key_mask=km)
    assert torch.equal(one, two)
    got = torch.autograd.grad(one, leaves, do)
    full = torch.autograd.grad(two, whole, do)
    for g, f, dim in zip(got, full, (0, 2, 1)):
        assert torch.equal(g, f.sum(dim, keepdim=True))
    x = q.detach().requires_grad_(True)                     # the same tensor three times, differentiated twice
    y = attention(x, x, x)
    a = torch.autograd.grad(y, x, y.detach(), retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, x, y.detach())[0])
    parts = [t.detach().clone().requires_grad_(True) for t in (q, q, q)]
    grads = torch.autograd.grad(attention(*parts), parts, y.detach())
    within(a, sum(g.double() for g in grads), 4 * half_step(dtype) * sum(g.double().abs() for g in grads), "shared")


# ------------------------------------------------------------------------------------------------ autograd, streams, graphs
def test_gradients_against_differences(dev):
    """<gradient, direction> of attention and of a gelu layer against central differences of the float64 formulas: the
    difference quotient of a smooth function is off by h^2 / 6 of its third derivative (some 1e-7 here), the gradients by
    1e-5 of their size at most."""
    from vista_amd.fused_tail import attention, linear_act
    q, k, v, km, do = make_attn((1, 9, 12, 2, 1, 2, 8, 8), F32, dev, 11, "some")
    x, w, b, r, dy = make_linear(9, 16, 12, F32, dev, 12, True, True)

    def attn64(q, k, v):
        K, V = k.transpose(1, 2).repeat_interleave(2, 1), v.transpose(1, 2)
        s = (q.transpose(1, 2) @ K.transpose(2, 3) * 8 ** -0.5).masked_fill(~km[:, None, None], -math.inf)
        return ((torch.softmax(s, -1) @ V).transpose(1, 2) * do.double()).sum()

    def lin64(x, w, b, r):
        return (torch.nn.functional.gelu(x @ w.t() + b + r) * dy.double()).sum()

    for args, f, g in (((q, k, v), attn64, lambda *a: (attention(*a, key_mask=km) * do).sum()),
                       ((x, w, b, r), lin64, lambda *a: (linear_act(*a, act="gelu") * dy).sum())):
        leaves = [a.clone().requires_grad_(True) for a in args]
        grads = torch.autograd.grad(g(*leaves), leaves)
        for i, grad in enumerate(grads):
            dirn = torch.randn(args[i].shape, dtype=torch.float64, device=dev)
            h = 1e-4
            at = [a.double() for a in args]
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + h * dirn, at[i] - h * dirn
            want = (f(*up) - f(*down)).item() / (2 * h)
            size = (grad.double().norm() * dirn.norm()).item()
            assert abs((grad.double() * dirn).sum().item() - want) <= 1e-5 * size + 1e-6, i


def test_autograd_returns_what_is_asked(dev):
    from vista_amd.fused_tail import attention, linear_act
    q, k, v, km, do = make_attn((2, 20, 30, 2, 2, 1, 16, 32), F32, dev, 1, "some")
    k.requires_grad_(True)
    out = attention(q, k, v, km)
    out.backward(do)
    assert k.grad is not None and q.grad is None
    with torch.no_grad():
        assert not attention(q, k, v, km).requires_grad
    x, w, b, r, dy = make_linear(6, 8, 10, F32, dev, 1, True, True)
    x3, r3 = x.view(2, 3, 8), r.view(2, 3, 10)
    w.requires_grad_(True)
    r3.requires_grad_(True)
    y = linear_act(x3, w, b, r3, "silu")
    assert y.shape == (2, 3, 10)
    y.backward(dy.view(2, 3, 10))
    assert w.grad.shape == w.shape and r3.grad.shape == r3.shape and b.grad is None
    out = attention(q, k, v, km)
    (gk,) = torch.autograd.grad(out.sum(), k, create_graph=True)
    with pytest.raises(RuntimeError):                      # once differentiable
        gk.sum().backward()


@pytest.mark.parametrize("shape", [(2, 200, 150, 4, 2, 1, 48, 96), (1, 70, 40, 2, 2, 1, 33, 50), (1, 3000, 60000, 1, 1, 1, 16, 24)])
def test_only_wanted_gradients_are_made(shape, dev):
    """Each subset of the three, from the plain call and through autograd: the bits of the full call, None for the others."""
    from vista_amd import ops
    from vista_amd.fused_tail import attention
    q, k, v, km, do = make_attn(shape, F32, dev, 1, "some")
    out, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    full = ops.attn_bwd(do, q, k, v, out, stats, km)
    calls = []
    real, ops._launch = ops._launch, lambda d, fn, *a: (calls.append((fn.__name__, a)), real(d, fn, *a))[1]
    try:
        for bits in range(8):
            want = [bool(bits >> i & 1) for i in range(3)]
            got = ops.attn_bwd(do, q, k, v, out, stats, km, None, *want)
            assert all((g is None) if not w else torch.equal(g, f) for g, f, w in zip(got, full, want))
            leaves = [t.clone().requires_grad_(w) for t, w in zip((q, k, v), want)]
            calls.clear()
            y = attention(*leaves, key_mask=km)
            assert y.requires_grad == any(want)
            if not any(want):
                continue
            y.backward(do)
            assert all((t.grad is None) if not w else torch.equal(t.grad, f) for t, f, w in zip(leaves, full, want))
            (args,) = [a for name, a in calls if "bwd" in name]
            assert [a is not None for a in args[12:15]] == want          # no room, and no work, for the others
    finally:
        ops._launch = real
    z = torch.zeros(2, 0, 2, 16, device=dev)
    q0 = torch.randn(2, 5, 2, 16, device=dev)
    o0, s0 = ops.attn_fwd(q0, z, z, want_stats=True)
    dq, dk, dv = ops.attn_bwd(torch.ones_like(o0), q0, z, z, o0, s0, want_dk=False)
    assert not dq.any() and dk is None and dv.shape == z.shape


def test_on_another_stream(dev):
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 200, 100, 2, 2, 1, 48, 96), F32, dev, 1, "some")
    want, stats = ops.attn_fwd(q, k, v, km, want_stats=True)
    grads = ops.attn_bwd(do, q, k, v, want, stats, km)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, st = ops.attn_fwd(q, k, v, km, want_stats=True)
        got = ops.attn_bwd(do, q, k, v, out, st, km)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, grads))


def test_captured_and_replayed(dev):
    """Forward and backward calls in one graph, another graph of the same calls beside it, replays on new inputs between eager work."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 130, 70, 2, 2, 1, 48, 96), F32, dev, 1, "some")
    x, w, b, r, dy = make_linear(700, 64, 96, F32, dev, 2, True, True)

    def step():
        out, st = ops.attn_fwd(q, k, v, km, want_stats=True)
        y, pre = ops.linear_fwd(x, w, b, r, "gelu", want_pre=True)
        return (out, *ops.attn_bwd(do, q, k, v, out, st, km), y, *ops.linear_bwd(dy, x, w, "gelu", pre))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            held = step()
        graphs.append((gr, held))
    gen = torch.Generator(device=dev).manual_seed(77)
    for i in range(4):
        for t in (q, k, v, do, x, dy):
            t.copy_(torch.randn(t.shape, generator=gen, device=dev))
        want = [t.clone() for t in step()]
        for gr, held in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_captured_and_replayed_bf16(dev):
    """The same with the rest of the output behind the statistics and g of a smooth activation in the workspace; two graphs, two streams."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 330, 170, 2, 2, 1, 48, 97), BF16, dev, 1, "some")
    x, w, b, r, dy = make_linear(700, 64, 96, BF16, dev, 2, True, True)

    def step():
        out, st = ops.attn_fwd(q, k, v, km, want_stats=True)
        y, pre = ops.linear_fwd(x, w, b, r, "silu", want_pre=True)
        return (out, *ops.attn_bwd(do, q, k, v, out, st, km), y, *ops.linear_bwd(dy, x, w, "silu", pre))

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for side in streams:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            held = step()
        graphs.append((gr, held))
    gen = torch.Generator(device=dev).manual_seed(79)
    for i in range(4):
        for t in (q, k, v, do, x, dy):
            t.copy_(torch.randn(t.shape, generator=gen, device=dev))
        want = [t.clone() for t in step()]
        for side, (gr, held) in zip(streams, graphs):       # both at once
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                gr.replay()
        torch.cuda.synchronize()
        for gr, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_captured_training_step(dev):
    """Attention into a layer, differentiated by autograd inside a capture, on leaves that no eager graph knows; replays on new inputs
    between eager steps on copies of the leaves."""
    from vista_amd.fused_tail import attention, linear_act
    q, k, v, km, _ = make_attn((2, 70, 150, 2, 2, 1, 24, 48), F32, dev, 3, "some")
    _, w, b, _, dy = make_linear(140, 96, 64, F32, dev, 4, True, False)

    def step(q, k, v, w, b):
        leaves = [t.requires_grad_(True) for t in (q, k, v, w, b)]
        y = linear_act(attention(q, k, v, km).view(140, 96), w, b, act="silu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    inputs = [t.detach() for t in (q, k, v, w, b)]
    eager = lambda: [t.clone() for t in step(*(i.detach().clone() for i in inputs))]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        held = step(*(i.detach() for i in inputs))
    gen = torch.Generator(device=dev).manual_seed(78)
    for i in range(4):
        for t in (*inputs, dy):
            t.copy_(torch.randn(t.shape, generator=gen, device=dev))
        want = eager()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_two_streams_at_once(dev):
    """The same operands on two streams whose work overlaps: no call shares a workspace with another."""
    from vista_amd import ops
    q, k, v, km, do = make_attn((2, 500, 300, 2, 2, 1, 96, 192), BF16, dev, 5, "some")
    x, w, _, s, dy = make_linear(3000, 128, 96, BF16, dev, 6, False, True)

    def step():
        out, st = ops.attn_fwd(q, k, v, km, want_stats=True)
        return (out, *ops.attn_bwd(do, q, k, v, out, st, km), *ops.linear_bwd(dy, x, w, "relu", s))

    want = step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


def test_forward_over_reverse_and_compiled_callers(dev):
    """A tangent that reaches the backward pass is refused; a compiled caller runs the same kernels (or refuses, but never returns
    unwritten memory)."""
    from torch.autograd import forward_ad
    from vista_amd.fused_tail import attention, linear_act
    q, k, v, km, do = make_attn((2, 40, 30, 2, 2, 1, 16, 32), F32, dev, 1, "some")
    x, w, b, r, dy = make_linear(20, 16, 24, F32, dev, 1, True, True)
    for f, args, cot in ((lambda *a: attention(*a, key_mask=km), (q, k, v), do), (linear_act, (x, w, b, r), dy)):
        leaves = [a.clone().requires_grad_(True) for a in args]
        out = f(*leaves)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            torch.autograd.grad(out, leaves, forward_ad.make_dual(cot, torch.ones_like(cot)))
        with torch.no_grad():
            want = f(*args) * 2
            assert torch.equal(torch.compile(lambda *a: f(*a) * 2, backend="eager")(*args), want)


# ------------------------------------------------------------------------------------------------ the block
def block(dev, heads=1):
    from vista_amd import dense_tail as dt
    torch.manual_seed(3)
    m = dt.Cross_Attention_Decouple(48, 48, 48, heads, (40, 40), (10, 10), (40, 12), (10, 12), 64)
    bev, rv = torch.randn(3, 48, 40, 40), torch.randn(3, 48, 40, 12)
    return m, bev, rv


@pytest.mark.parametrize("heads", [1, 2])
def test_fused_block_runs_the_operators_together(heads, dev):
    """The neck with its attention block on the kernels against the stock module in float64, outputs and every gradient: 1e-4 of
    each tensor's largest value, the bar of this path's fp32 parity."""
    from vista_amd.fused_tail import FusedConvAttention, FusedFeedForward, fuse_cross_attention
    m, bev, rv = block(dev, heads)
    import copy
    stock = copy.deepcopy(m).double()
    keys = list(m.state_dict())
    fused = fuse_cross_attention(m).to(dev)
    assert list(fused.state_dict()) == keys
    kinds = [type(c) for c in fused.modules()]
    assert kinds.count(FusedConvAttention) == 1 and kinds.count(FusedFeedForward) == 2
    bev64, rv64 = bev.double().requires_grad_(True), rv.double().requires_grad_(True)
    bevg, rvg = bev.to(dev).requires_grad_(True), rv.to(dev).requires_grad_(True)
    want, _ = stock((bev64, rv64), need_maps=False)
    got, maps = fused((bevg, rvg), need_maps=False)
    assert maps == [None, None]
    cot = [torch.randn(t.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)) for i, t in enumerate(want)]
    sum((w * c).sum() for w, c in zip(want, cot)).backward()
    sum((g * c.float().to(dev)).sum() for g, c in zip(got, cot)).backward()

    def close(a, b, what):
        err = (a.detach().cpu().double() - b.detach()).abs().max().item() / max(b.detach().abs().max().item(), 1e-12)
        assert err <= 1e-4, (what, err)

    for g, w in zip(got, want):
        close(g, w, "out")
    close(bevg.grad, bev64.grad, "bev")
    close(rvg.grad, rv64.grad, "rv")
    for (name, a), (_, b) in zip(fused.named_parameters(), stock.named_parameters()):
        if ".k_" in name and name.endswith("bias"):        # softmax is blind to a shift of a query's scores: exactly zero
            assert a.grad.abs().max().item() <= 1e-4 * b.grad.abs().max().clamp(min=1.0).item(), name
        else:
            close(a.grad, b.grad, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_fused_neck_at_full_size(dtype, dev):
    """The detector's own neck (1600 queries over 480 keys, 384 channels, one head): the fused block and the stock one on the same
    maps. fp32: 1e-4 of the largest value; bf16: sixteen roundings of half a step (2^-8) of it lie between a map and the same map."""
    from vista_amd.dense_tail import Cross_Attention_Decouple
    from vista_amd.fused_tail import fuse_cross_attention
    import copy
    torch.manual_seed(7)
    stock = Cross_Attention_Decouple(384, 384, 384, 1, (160, 160), (40, 40), (160, 12), (40, 12), 512).eval().to(dev)
    fused = fuse_cross_attention(copy.deepcopy(stock)).to(dtype)
    bev, rv = torch.randn(2, 384, 160, 160, device=dev), torch.randn(2, 384, 160, 12, device=dev)
    with torch.no_grad():
        want, _ = stock((bev, rv), need_maps=False)
        got, _ = fused((bev.to(dtype), rv.to(dtype)), need_maps=False)
    for a, b in zip(got, want):
        tol = 1e-4 if dtype == F32 else 16 * 2.0 ** -8
        assert a.dtype == dtype and (a.float() - b).abs().max() <= tol * b.abs().max()


def test_fused_block_with_maps_runs_the_stock_path(dev):
    from vista_amd.fused_tail import fuse_cross_attention
    m, bev, rv = block(dev)
    m, bev, rv = m.to(dev).eval(), bev.to(dev), rv.to(dev)
    with torch.no_grad():
        want, maps = m((bev, rv))
        layer = m.cross_atten.cross_atten
        fuse_cross_attention(m)
        blk = m.cross_atten.cross_atten
        assert blk is not layer and blk.q_sem_conv is layer.q_sem_conv
        q = torch.randn(2, 48, 5, 5, device=dev)
        kv = torch.randn(2, 48, 5, 3, device=dev)
        a, ma = layer(q, kv, kv)
        b, mb = blk(q, kv, kv)
        assert all(torch.equal(x, y) for x, y in zip(a + ma, b + mb))
        mask = torch.ones(2, 15, dtype=torch.bool, device=dev)
        c, none = blk(q, kv, kv, need_maps=False, key_mask=mask)
        assert none == [None, None] and torch.equal(c[0], blk(q, kv, kv, need_maps=False)[0][0])
        with pytest.raises(ValueError):
            blk(q, kv, kv, key_mask=mask)


def test_fused_layers_return_the_layout_of_the_stock_ones(dev):
    """Tokens [HW, B, C], contiguous: a caller's .view() works on them; a feed-forward layer of transposed tokens likewise."""
    from vista_amd.dense_tail import ConvAttentionLayer_Decouple, FeedFowardLayer
    from vista_amd.fused_tail import fuse_cross_attention
    att, ffn = ConvAttentionLayer_Decouple(24, 2).to(dev), FeedFowardLayer(24, 40).to(dev)
    fatt, fffn = fuse_cross_attention(att), fuse_cross_attention(ffn)
    q, kv = torch.randn(3, 24, 5, 4, device=dev), torch.randn(3, 24, 2, 7, device=dev)
    for a, b in zip(att(q, kv, kv, need_maps=False)[0], fatt(q, kv, kv, need_maps=False)[0]):
        assert b.shape == a.shape and b.stride() == a.stride() and b.is_contiguous()
        within(b, a.double(), 1e-4 * a.abs().max().double().expand_as(a), "tokens")
        for v in (b, b.transpose(0, 1), b[:, :1]):
            y, z = ffn(v), fffn(v)
            assert z.stride() == y.stride()
            within(z, y.double(), 1e-4 * y.abs().max().double().expand_as(y), "ffn")


@pytest.mark.parametrize("half", [BF16, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
def test_fused_block_under_autocast(half, masked, dev):
    """The stock block runs under autocast, so the fused one does: outputs and gradients against the block in float64, no farther than the
    stock block's own and sixteen roundings of half a bf16 step of the largest value. Autocast to float16 runs the stock form."""
    import copy
    from vista_amd.dense_tail import CrossAttenBlock_Decouple
    from vista_amd.fused_tail import fuse_cross_attention
    torch.manual_seed(5)
    stock = CrossAttenBlock_Decouple(48, 2, 64).to(dev)
    fused = fuse_cross_attention(copy.deepcopy(stock))
    exact = copy.deepcopy(stock).double()
    bev, rv = torch.randn(3, 48, 10, 9, device=dev), torch.randn(3, 48, 10, 4, device=dev)
    if masked:                                             # the layer's own argument: a stock layer has none
        km = torch.rand(3, 40, device=dev) > 0.3
        with torch.autocast("cuda", half):
            if half == BF16:
                a = fused.cross_atten(bev, rv, rv, need_maps=False, key_mask=km)[0]
            else:
                with pytest.raises(ValueError, match="key_mask"):
                    fused.cross_atten(bev, rv, rv, need_maps=False, key_mask=km)
                return
        for x, y in zip(a, fused.cross_atten(bev, rv, rv, need_maps=False, key_mask=km)[0]):
            assert x.dtype == F32 and (x - y).abs().max() <= 16 * 2.0 ** -8 * y.abs().max()
        return
    cot = [torch.randn(3, 48, 10, 9, device=dev) for _ in range(2)]

    def step(m, cast):
        dt = next(m.parameters()).dtype
        x, y = (t.to(dt).requires_grad_(True) for t in (bev, rv))
        with torch.autocast("cuda", half, enabled=cast):
            out, _ = m(x, y, need_maps=False)
        got = torch.autograd.grad(out, (x, y), [c.to(o.dtype) for c, o in zip(cot, out)], retain_graph=True)
        par = torch.autograd.grad(out, list(m.parameters()), [c.to(o.dtype) for c, o in zip(cot, out)])
        return [(o.detach().dtype, o.detach().double()) for o in (*out, *got, *par)]

    names = ["sem", "geo", "bev", "rv"] + [n for n, _ in stock.named_parameters()]
    for name, (t, a), (u, b), (_, c) in zip(names, step(fused, True), step(stock, True), step(exact, False)):
        assert t == u, name
        size = c.abs().max().clamp(min=1.0 if ".k_" in name else 0.0)            # (gradients of the biases of k are exactly zero)
        if half == BF16:
            assert (a - c).abs().max() <= (b - c).abs().max() + 16 * 2.0 ** -8 * size, name
        else:
            assert (a - b).abs().max() <= 2.0 ** -8 * size, name


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(dev):
    from vista_amd import ops
    from vista_amd._lib import VxError
    z = lambda *s, dtype=F32, device=dev: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    q, k, v = z(2, 3, 4, 8), z(2, 5, 2, 8), z(2, 5, 1, 16)
    bad = [dict(q=z(2, 3, 4, 8, dtype=torch.float16)), dict(k=z(2, 5, 2, 8, dtype=BF16)), dict(k=z(2, 5, 3, 8)), dict(k=z(2, 5, 2, 9)),
           dict(k=z(2, 6, 2, 8)), dict(k=z(1, 5, 2, 8)), dict(q=z(2, 3, 8)), dict(q=z(2, 3, 4, 193), k=z(2, 5, 2, 193)),
           dict(v=z(2, 5, 1, 385)), dict(v=z(2, 5, 0, 16)), dict(q=z(2, 3, 4, 0), k=z(2, 5, 2, 0)),
           dict(key_mask=z(2, 5)), dict(key_mask=z(2, 4, dtype=torch.bool)), dict(key_mask=z(2, 1, 1, 5, dtype=torch.bool))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.attn_fwd(**dict(dict(q=q, k=k, v=v), **kw))
    with pytest.raises(VxError):
        ops.attn_fwd(q, k.cpu(), v)
    out, stats = ops.attn_fwd(q, k, v, want_stats=True)
    for kw in (dict(dout=z(2, 3, 4, 8)), dict(dout=z(2, 3, 4, 16, dtype=BF16)), dict(out=z(2, 4, 3, 16).transpose(1, 2)),
               dict(stats=stats[:1]), dict(stats=stats.double())):
        with pytest.raises(ValueError):
            ops.attn_bwd(**dict(dict(dout=out, q=q, k=k, v=v, out=out, stats=stats), **kw))
    x, w = z(4, 6), z(5, 6)
    for kw in (dict(act="tanh"), dict(act=None), dict(weight=z(5, 7)), dict(x=z(4, 6, dtype=torch.float64)), dict(bias=z(6)),
               dict(bias=z(5, dtype=BF16)), dict(residual=z(4, 6)), dict(residual=z(1, 5)), dict(x=z(2, 4, 6)), dict(x=z(4, 0), weight=z(5, 0))):
        with pytest.raises(ValueError):
            ops.linear_fwd(**dict(dict(x=x, weight=w), **kw))
    for kw in (dict(act="relu"), dict(act="gelu", saved=z(4, 6)), dict(dy=z(5, 4)), dict(act="swish", saved=z(4, 5))):
        with pytest.raises(ValueError):
            ops.linear_bwd(**dict(dict(dy=z(4, 5), x=x, weight=w), **kw))
