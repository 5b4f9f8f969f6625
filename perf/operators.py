"""Cross-view attention and the dense layers around it: what is timed of vista_amd.fused_tail / vista_amd.ops.

Four operators, each as a program of this framework calls it:
  attn         softmax(scale q k^T) v with a key mask, no gradients (inference of the cross-view neck)
  attn_grad    the same inside a training step: output and the gradients of q, k and v
  linear       act(x w^T + bias + residual) (the neck's 1x1 convolutions and feed-forward layers)
  linear_grad  the backward pass of one such layer from what its forward pass saved

Layouts: q [batch, q_len, heads, dim], k [batch, k_len, k_heads, dim], v [batch, k_len, v_heads, v_dim]; query head h reads
key head h // (heads / k_heads) and value head h // (heads / v_heads). The neck's semantic and geometric read-outs are two
query / key heads over one value head. x [rows, fin], weight [fout, fin].
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_ACTS = ("none", "relu", "gelu", "silu")


# ------------------------------------------------------------------------------------------------ cases
def _attn(name, op, dtype, batch, q_len, k_len, heads, k_heads, v_heads, dim, v_dim, mask):
    c = dict(op=op, dtype=dtype, batch=batch, q_len=q_len, k_len=k_len, heads=heads, k_heads=k_heads, v_heads=v_heads,
             dim=dim, v_dim=v_dim, mask=mask)
    return dict(c, name=name) if name else c


def _lin(name, op, dtype, rows, fin, fout, act, bias, residual):
    c = dict(op=op, dtype=dtype, rows=rows, fin=fin, fout=fout, act=act, bias=bias, residual=residual)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one query token over the RV blocks of one frame: a single anchor re-read, latency only
        _attn("attn one token", "attn", "f32", 1, 1, 480, 2, 2, 1, 192, 384, "none"),
        # the VISTA neck: 40 x 40 BEV blocks over 40 x 12 RV blocks, embed 384, 1 head, two read-outs of one value map,
        # 4 frames, blocks without a return masked
        _attn("attn vista blocks b4", "attn", "f32", 4, 1600, 480, 2, 2, 1, 192, 384, "blocks"),
        # the same neck without the block pooling: every BEV cell over every RV cell of one frame, bf16 inference
        _attn("attn full maps bf16", "attn", "bf16", 1, 25600, 1920, 2, 2, 1, 192, 384, "blocks"),
        # ordinary multi-head self-attention over a frame's occupied blocks, an odd number of them
        _attn("attn self 2037 bf16", "attn", "bf16", 2, 2037, 2037, 8, 8, 8, 48, 48, "none"),
        # training step of the neck at the batch size of the shipped training run
        _attn("grad vista blocks b4", "attn_grad", "f32", 4, 1600, 480, 2, 2, 1, 192, 384, "blocks"),
        # four heads, shared key heads, ragged sizes, a batch in which one frame has no key at all
        _attn("grad ragged bf16", "attn_grad", "bf16", 3, 777, 301, 4, 2, 1, 96, 192, "blank"),
        # training on unpooled maps, one frame: the largest case
        _attn("grad full maps", "attn_grad", "f32", 1, 25600, 1920, 2, 2, 1, 192, 384, "blocks"),
        # a feed-forward layer on a handful of tokens
        _lin("linear 7 rows", "linear", "f32", 7, 384, 512, "relu", True, False),
        # out convolution + identity of the neck, 4 frames of 1600 blocks
        _lin("linear out conv b4", "linear", "f32", 6400, 384, 384, "none", True, True),
        # first feed-forward layer on every BEV cell of 8 frames, bf16
        _lin("linear ffn maps bf16", "linear", "bf16", 204800, 384, 512, "relu", True, False),
        # backward of the second feed-forward layer, 4 frames of blocks
        _lin("lingrad ffn2 b4", "linear_grad", "f32", 6400, 512, 384, "none", True, True),
        # backward of the first one on every BEV cell of 4 frames, odd row count
        _lin("lingrad ffn1 bf16", "linear_grad", "bf16", 102399, 384, 512, "relu", True, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn_grad", "linear", "linear_grad"])
    dtype = rng.choice(["f32", "bf16"])
    if op.startswith("attn"):
        kind = rng.choice(["neck", "neck", "self", "odd"])
        if kind == "neck":                      # embed 384 over n heads, keys half as wide as values
            n = rng.choice([1, 2, 4, 8])
            heads, k_heads, v_heads, dim, v_dim = 2 * n, 2 * n, n, 192 // n, 384 // n
        elif kind == "self":
            v_heads = rng.choice([1, 2, 4])
            heads = v_heads * rng.choice([1, 2, 3])
            k_heads, dim = v_heads, 8 * rng.randint(2, 16)
            v_dim = dim
        else:
            v_heads = k_heads = rng.randint(1, 3)
            heads = k_heads * rng.randint(1, 2)
            dim, v_dim = rng.randint(5, 192), rng.randint(5, 384)
        batch = rng.randint(1, 6)
        q_len = _log(rng, 1, 25600)
        top = 25600 * 1920 * 2 * 576            # no dearer than the largest listed case
        k_top = max(1, min(8192, top // (batch * heads * q_len * (dim + v_dim))))
        # over one key the gradients of q and k are zero and every computed value is rounding: 16 keys and more there
        k_len = _log(rng, 16, max(16, k_top)) if op == "attn_grad" else _log(rng, 1, k_top)
        return _attn(None, op, dtype, batch, q_len, k_len, heads, k_heads, v_heads, dim, v_dim,
                     rng.choice(["none", "blocks", "blank"] if batch > 1 else ["none", "blocks"]))
    rows = _log(rng, 1, 204800)
    fin, fout = (rng.choice([64, 128, 384, 512, 640]) if rng.random() < 0.6 else rng.randint(5, 700) for _ in range(2))
    if rows * fin * fout > 102400 * 384 * 512:
        rows = 102400 * 384 * 512 // (fin * fout)
    return _lin(None, op, dtype, rows, fin, fout, rng.choice(_ACTS), rng.random() < 0.8, rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def rnd(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dt)

    s = dict(case)
    if case["op"].startswith("attn"):
        b, h, d, dv = case["batch"], case["heads"], case["dim"], case["v_dim"]
        s["q"], s["k"] = rnd(b, case["q_len"], h, d), rnd(b, case["k_len"], case["k_heads"], d)
        s["v"] = rnd(b, case["k_len"], case["v_heads"], dv)
        s["key_mask"] = None
        if case["mask"] != "none":              # about a third of the RV blocks hold no return
            s["key_mask"] = torch.rand((b, case["k_len"]), generator=g, device="cuda") > 0.35
            s["key_mask"][:, 0] = True
            if case["mask"] == "blank":         # a frame without any return
                s["key_mask"][0] = False
        if case["op"] == "attn_grad":
            s["dout"] = rnd(b, case["q_len"], h, dv)
            for t in ("q", "k", "v"):
                s[t].requires_grad_(True)
        return s
    m, k, n = case["rows"], case["fin"], case["fout"]
    s["x"], s["weight"] = rnd(m, k), rnd(n, k, std=k ** -0.5)
    if case["op"] == "linear":
        s["bias"] = rnd(n, std=0.1) if case["bias"] else None
        s["residual"] = rnd(m, n) if case["residual"] else None
    else:
        s["dy"] = rnd(m, n)
        pre = rnd(m, n)                         # what the forward pass saved: its sum before the activation, or relu's output
        s["saved"] = {"none": None, "relu": pre.clamp(min=0), "gelu": pre, "silu": pre}[case["act"]]
    return s


# ------------------------------------------------------------------------------------------------ the pass
def _plain_attention(s, grad):
    dt = s["q"].dtype
    q, k, v = (s[t].detach().float().transpose(1, 2) for t in ("q", "k", "v"))     # [batch, heads, len, dim]
    h, b = q.shape[1], q.shape[0]
    gk, gv = h // k.shape[1], h // v.shape[1]
    mask = s["key_mask"]
    if mask is not None:                       # a masked key has no part in anything, whatever it holds
        dead = ~mask[:, None, :, None]
        k, v = k.masked_fill(dead, 0), v.masked_fill(dead, 0)
    k, v = k.repeat_interleave(gk, 1), v.repeat_interleave(gv, 1)
    scale = q.shape[-1] ** -0.5
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    if mask is not None:
        p.masked_fill_(~mask[:, None, None, :], -math.inf)
    p = torch.exp(p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)))
    p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))                             # a row without keys: 0
    out = torch.matmul(p, v)
    if not grad:
        return out.transpose(1, 2).to(dt).contiguous()
    do = s["dout"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dk = dk.view(b, h // gk, gk, *dk.shape[2:]).sum(2)
    dv = dv.view(b, h // gv, gv, *dv.shape[2:]).sum(2)
    return {n: t.transpose(1, 2).to(dt).contiguous() for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv))}


def _plain_linear(s):
    y = torch.matmul(s["x"].float(), s["weight"].float().t())
    if s["bias"] is not None:
        y += s["bias"].float()
    if s["residual"] is not None:
        y += s["residual"].float()
    if s["act"] == "relu":
        y = y.clamp_(min=0)
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["x"].dtype)


def _plain_linear_grad(s):
    dt, g = s["dy"].dtype, s["dy"].float()
    if s["act"] == "relu":
        g = g * (s["saved"] > 0)
    elif s["act"] == "gelu":
        a = s["saved"].float()
        g = g * (0.5 * (1 + torch.erf(a * math.sqrt(0.5))) + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi)))
    elif s["act"] == "silu":
        a = s["saved"].float()
        e = 1 / (1 + torch.exp(-a))
        g = g * (e * (1 + a * (1 - e)))
    r = {"dx": torch.matmul(g, s["weight"].float()), "dw": torch.matmul(g.t().contiguous(), s["x"].float())}
    if s["bias"]:
        r["dbias"] = g.sum(0)
    if s["residual"]:
        r["dresidual"] = g
    return {n: t.to(dt) for n, t in r.items()}


def run(state):
    s = state
    if not own:
        if s["op"].startswith("attn"):
            return _plain_attention(s, s["op"] == "attn_grad")
        return _plain_linear(s) if s["op"] == "linear" else _plain_linear_grad(s)
    from vista_amd import fused_tail, ops
    if s["op"] == "attn":
        return fused_tail.attention(s["q"], s["k"], s["v"], key_mask=s["key_mask"])
    if s["op"] == "attn_grad":
        out = fused_tail.attention(s["q"], s["k"], s["v"], key_mask=s["key_mask"])
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if s["op"] == "linear":
        return fused_tail.linear_act(s["x"], s["weight"], s["bias"], s["residual"], act=s["act"])
    dx, dw, db, dres = ops.linear_bwd(s["dy"], s["x"], s["weight"], act=s["act"], saved=s["saved"], want_dbias=s["bias"])
    r = {"dx": dx, "dw": dw}
    if s["bias"]:
        r["dbias"] = db
    if s["residual"]:
        r["dresidual"] = dres
    return r


# ------------------------------------------------------------------------------------------------ work and truth
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("attn"):
        b, sq, sk, h, d, dv = (case[t] for t in ("batch", "q_len", "k_len", "heads", "dim", "v_dim"))
        nq, nk, nv, no = b * sq * h * d, b * sk * case["k_heads"] * d, b * sk * case["v_heads"] * dv, b * sq * h * dv
        mask = 0 if case["mask"] == "none" else b * sk
        pair = 2 * b * h * sq * sk
        if case["op"] == "attn":
            return {"bytes": e * (nq + nk + nv + no) + mask, "flops": pair * (d + dv)}
        # forward, then scores again, dP, dV, dK, dQ
        return {"bytes": e * (2 * (nq + nk + nv) + 2 * no) + mask, "flops": pair * (d + dv + 3 * d + 2 * dv)}
    m, k, n = case["rows"], case["fin"], case["fout"]
    if case["op"] == "linear":
        return {"bytes": e * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    maps = 1 + (case["act"] != "none") + bool(case["residual"])
    return {"bytes": e * (2 * m * k + 2 * n * k + maps * m * n + (n if case["bias"] else 0)), "flops": 4 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"].startswith("attn"):
        q, k, v = s["q"].detach(), s["k"].detach(), s["v"].detach()
        (b, sq, h, d), sk, dv = q.shape, k.shape[1], v.shape[3]
        gk, gv, scale = h // k.shape[2], h // v.shape[2], 1.0 / math.sqrt(d)
        grad = case["op"] == "attn_grad"
        out = torch.zeros((b, sq, h, dv), dtype=f8, device="cuda")
        dq, dk, dvv = (torch.zeros(t.shape, dtype=f8, device="cuda") for t in (q, k, v))
        for i in range(b):
            live = torch.arange(sk, device="cuda") if s["key_mask"] is None else torch.nonzero(s["key_mask"][i])[:, 0]
            if not live.numel():
                continue
            for j in range(h):
                kk, vv = k[i, live, j // gk].to(f8), v[i, live, j // gv].to(f8)
                for lo in range(0, sq, 4096):
                    qq = q[i, lo:lo + 4096, j].to(f8)
                    w = torch.softmax(scale * (qq @ kk.t()), 1)
                    o = w @ vv
                    out[i, lo:lo + 4096, j] = o
                    if grad:
                        go = s["dout"][i, lo:lo + 4096, j].to(f8)
                        t = w * (go @ vv.t() - (go * o).sum(1)[:, None]) * scale
                        dq[i, lo:lo + 4096, j] = t @ kk
                        dk[i, :, j // gk].index_add_(0, live, t.t() @ qq)
                        dvv[i, :, j // gv].index_add_(0, live, w.t() @ go)
        return {"out": out, "dq": dq, "dk": dk, "dv": dvv} if grad else out
    x, w = s["x"].to(f8), s["weight"].to(f8)
    if case["op"] == "linear":
        y = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].to(f8))
        if s["residual"] is not None:
            y = y + s["residual"].to(f8)
        f = torch.nn.functional
        return {"none": lambda t: t, "relu": torch.relu, "gelu": f.gelu, "silu": f.silu}[case["act"]](y)
    g = s["dy"].to(f8)
    if case["act"] == "relu":
        g = torch.where(s["saved"] > 0, g, torch.zeros_like(g))
    elif case["act"] != "none":
        a = s["saved"].to(f8)
        if case["act"] == "gelu":
            slope = torch.special.ndtr(a) + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
        else:
            slope = torch.sigmoid(a) * (1 + a * torch.sigmoid(-a))
        g = g * slope
    r = {"dx": g @ w, "dw": g.t() @ x}
    if case["bias"]:
        r["dbias"] = g.sum(0)
    if case["residual"]:
        r["dresidual"] = g
    return r
