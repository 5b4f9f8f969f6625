"""The cross-view attention block of the dense tail on hand-written kernels, forward and backward.

`attention` and `linear_act` are differentiable torch functions over the libvx kernels of vista_amd/csrc/vx_attn.hip and
vx_linear.hip (HIP tensors, float32 or bfloat16, no CPU path); `fuse_cross_attention(module)` rewrites the
ConvAttentionLayer_Decouple and FeedFowardLayer of a module to run on them:
  attention   det3d/models/necks/attention.py:55-124   both read-outs as two query / key heads over one value head
  linear_act  attention.py:36-41 (1x1 value / out convolutions, identity added in the epilogue), :127-146 (feed-forward)
Gradients are exact formulas of the saved tensors (once differentiable). Both run on the caller's stream, allocate through
torch's caching allocator only, and can be captured in a HIP graph; before a backward pass is captured, drop every eager graph of
the same leaves (torch ties a leaf's gradient accumulation to the stream on which it was first seen).
"""
import torch
from torch import nn

from . import _lib, ops
from .dense_tail import ConvAttentionLayer_Decouple, FeedFowardLayer


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale):
        q, k, v, key_mask, geo = ops._attn_args(q, k, v, key_mask)
        out, stats = ops._attn_fwd_run(q, k, v, key_mask, geo, scale, True)
        ctx.save_for_backward(q, k, v, key_mask, out, stats)
        ctx.geo, ctx.scale = geo, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, key_mask, out, stats = ctx.saved_tensors
        ops._check_seen(dout)        # (out's shape, dtype and device: the engine sees to that)
        dq, dk, dv = ops._attn_bwd_run(dout, q, k, v, key_mask, ctx.geo, out, stats, ctx.scale, ctx.needs_input_grad[:3])
        return dq, dk, dv, None, None


def attention(q, k, v, key_mask=None, scale=None):
    """softmax(scale q k^T) v. q [b, sq, heads, dim], k [b, sk, k_heads, dim], v [b, sk, v_heads, v_dim] -> [b, sq, heads, v_dim];
    key and value heads are shared by consecutive query heads. key_mask: bool [b, sk], True where the key takes part; a masked key
    has no part in the output or any gradient, whatever it holds, and a query without keys gives zeros. scale defaults to
    dim ** -0.5; dim <= 192, v_dim <= 384."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFn.apply(q, k, v, key_mask, scale)
    return ops.attn_fwd(q, k, v, key_mask, scale)[0]


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, pre = ops.linear_fwd(x, weight, bias, residual, act, want_pre=act in ("gelu", "silu"))
        ctx.save_for_backward(x, weight, y if act == "relu" else pre)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db, dpre = ops.linear_bwd(dy, x, weight, ctx.act, saved, *need[:3])
        return dx, dw, db, dpre if need[3] else None, None


def linear_act(x, weight, bias=None, residual=None, act="none"):
    """act(x w^T + bias + residual) over the last dimension of x [..., fin]; weight [fout, fin], bias [fout], residual
    [..., fout]. act: none, relu, gelu (erf form), silu; it comes after the residual, as in the sparse convolutions' epilogue."""
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                        or (residual is not None and residual.requires_grad))
    if x.dim() == 2:
        return _LinearFn.apply(x, weight, bias, residual, act) if grad else ops.linear_fwd(x, weight, bias, residual, act)[0]
    if x.dim() < 1 or (residual is not None and residual.shape[:-1] != x.shape[:-1]):
        raise ValueError("x must be [..., fin] and residual [..., fout] with the same leading dimensions")
    x2 = x.reshape(-1, x.shape[-1])
    r2 = residual.reshape(-1, residual.shape[-1]) if residual is not None else None
    y = _LinearFn.apply(x2, weight, bias, r2, act) if grad else ops.linear_fwd(x2, weight, bias, r2, act)[0]
    return y.view(*x.shape[:-1], weight.shape[0])


def _hooked(module):
    return bool(module._forward_pre_hooks or module._forward_hooks or module._backward_pre_hooks or module._backward_hooks)


def _plain_conv1x1(m):
    return (isinstance(m, nn.Conv2d) and type(m).forward is nn.Conv2d.forward and m.kernel_size == (1, 1) and m.stride == (1, 1)
            and m.padding == (0, 0) and m.groups == 1)


def _plain_linear(m):
    return isinstance(m, nn.Linear) and type(m).forward is nn.Linear.forward


def _become(module, layer):
    """All that `layer` holds -- submodules (one that stands under two names too), parameters and buffers of its own, training flags,
    attributes -- in containers of `module`'s own."""
    module.__dict__.update((k, v.copy() if isinstance(v, (dict, set)) else v) for k, v in layer.__dict__.items())


def _autocast():
    """The type that autocast asks for, or None outside of it."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None


def _layer(x, weight, bias, residual=None, act="none"):
    """linear_act as one of autocast's operators: its product in bfloat16 there, the residual added in its own type."""
    if _autocast() is None:
        return linear_act(x, weight, bias, residual, act)
    half = [t.to(torch.bfloat16) if t is not None else None for t in (x, weight, bias)]
    y = linear_act(*half, act=act)
    return y if residual is None else residual + y


def _conv1x1(conv, x, residual=None):
    """A 1x1 nn.Conv2d over tokens [..., c] instead of a map [b, c, h, w]."""
    return _layer(x, conv.weight.flatten(1), conv.bias, residual)


class FusedConvAttention(nn.Module):
    """ConvAttentionLayer_Decouple on `attention` and `linear_act`; shares the layer's submodules, so parameters and
    state_dict keys are the layer's. The attention maps are not formed: need_maps=True runs the layer's own forward, and so do hooks on
    a submodule of `direct`, whose weight is read without a call of it (weight_norm, prune and the like make the weight in a hook), and
    a submodule there that is no 1x1 convolution."""

    direct = ("v_conv", "out_sem_conv", "out_geo_conv")

    @classmethod
    def computes(cls, layer):
        """Whether the kernels can stand in for the layer's own forward."""
        return (all(_plain_conv1x1(getattr(layer, name, None)) for name in cls.direct) and layer.head_dim <= _lib.VX_ATTN_MAX_DIM
                and layer.v_conv.out_channels // layer.numhead <= _lib.VX_ATTN_MAX_VDIM)

    def __init__(self, layer):
        _become(self, layer)

    def forward(self, query, key, value, q_pos_emb=None, k_pos_emb=None, need_maps=True, key_mask=None):
        """-> ([tokens[HW_q, B, C]] x2, [None, None]); key_mask bool [B, HW_kv], True where the key block takes part."""
        if need_maps or not _direct(self):
            if key_mask is not None:
                raise ValueError("key_mask is supported without attention maps (need_maps=False) and where the kernels compute the "
                                 f"layer (no hooks on {', '.join(self.direct)}) only")
            return ConvAttentionLayer_Decouple.forward(self, query, key, value, q_pos_emb, k_pos_emb, need_maps)
        identity = query
        if q_pos_emb is not None:
            query = query + q_pos_emb
        if k_pos_emb is not None:
            shared = value is key            # the embedding reaches the value path too (attention.py:64-65, :206)
            key = key + k_pos_emb
            if shared:
                value = key
        b, c, hq, wq = identity.shape
        n, sq = self.numhead, hq * wq

        def tokens(t):                       # [B, c, H, W] -> [B, H*W, c]
            return t.flatten(2).transpose(1, 2).contiguous()

        def heads(sem, geo):                 # two maps -> [B, H*W, 2 n, d], a head's read-outs side by side
            s = torch.stack([sem.flatten(2), geo.flatten(2)], 1).view(b, 2, n, self.head_dim, -1)
            return s.permute(0, 4, 2, 1, 3).reshape(b, -1, 2 * n, self.head_dim)

        v = _conv1x1(self.v_conv, tokens(value)).view(b, -1, n, c // n)
        r = attention(heads(self.q_sem_conv(query), self.q_geo_conv(query)), heads(self.k_sem_conv(key), self.k_geo_conv(key)),
                      v, key_mask, float(self.head_dim) ** -0.5).view(b, sq, n, 2, c // n)
        rows = identity.flatten(2).permute(2, 0, 1).contiguous()
        outs = []
        for i, (conv, norm) in enumerate(((self.out_sem_conv, self.sem_norm), (self.out_geo_conv, self.geo_norm))):
            outs.append(norm(_conv1x1(conv, r[:, :, :, i].transpose(0, 1).reshape(sq, b, c), rows)))
        return outs, [None, None]


class FusedFeedForward(nn.Module):
    """FeedFowardLayer on `linear_act`: ReLU in the first product's epilogue, the residual in the second's. Hooks on a submodule of
    `direct`, or another kind of submodule there: the layer's own forward, which calls them."""

    direct = ("linear1", "linear2", "activation")

    @classmethod
    def computes(cls, layer):
        act = getattr(layer, "activation", None)
        return all(_plain_linear(getattr(layer, name, None)) for name in cls.direct[:2]) and type(act) is nn.ReLU

    def __init__(self, layer):
        _become(self, layer)

    def forward(self, view):
        if not _direct(self):
            return FeedFowardLayer.forward(self, view)
        h = _layer(view, self.linear1.weight, self.linear1.bias, act="relu")
        return self.norm(_layer(h, self.linear2.weight, self.linear2.bias, view))


def _direct(fused):
    return fused.computes(fused) and _autocast() in (None, torch.bfloat16) and not any(_hooked(fused._modules[name]) for name in fused.direct)


_SWAP = {ConvAttentionLayer_Decouple: FusedConvAttention, FeedFowardLayer: FusedFeedForward}


def _fusable(module):
    return type(module) in _SWAP and _SWAP[type(module)].computes(module)


def fuse_cross_attention(module):
    """Rewrite `module` in place: every ConvAttentionLayer_Decouple and FeedFowardLayer in it runs on the fused kernels
    (inference and training; HIP tensors only from then on, unless attention maps are asked for). Parameters, buffers and
    state_dict keys are unchanged. A layer with hooks, or with hooks on a submodule that the fused form does not call, is refused before
    anything is changed; hooks that such a submodule gets later run the layer's own forward. A layer that the kernels do not compute
    (heads wider than `attention` takes, another activation, submodules of another kind) is left as it is. Under autocast to bfloat16
    the products run in bfloat16, under another autocast the layer's own forward does. Returns `module`, or its replacement
    when it is such a layer itself."""
    for name, layer in module.named_modules():
        if _fusable(layer):
            for at, m in [("", layer)] + [("." + c, layer._modules[c]) for c in _SWAP[type(layer)].direct]:
                if _hooked(m):
                    raise ValueError(f"{name or type(layer).__name__}{at} has hooks, which the fused layer would not call")
    return _rewrite(module, {})


def _rewrite(module, done):
    """`done`: layer -> its replacement, for layers that stand in several places."""
    if _fusable(module):
        if module not in done:
            done[module] = _SWAP[type(module)](module)
        return done[module]
    for name, child in list(module._modules.items()):
        if child is not None:
            module._modules[name] = _rewrite(child, done)
    return module
