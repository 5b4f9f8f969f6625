"""CPU: refusals of the attention and dense-layer entry points, at the C-ABI (no launch happens) and in Python."""
import ctypes

import pytest
import torch

from vista_amd import _lib, dense_tail, fused_tail, ops

ERR_ARG, ERR_WS = -1, -3
FAKE = ctypes.c_void_p(256)          # never read: every call below is refused before a launch


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def fwd(shape, strides=(1,) * 10, q=FAKE, out=FAKE, dtype=0, ws=FAKE, wsb=1 << 40):
    return _lib.lib().vx_attn_fwd(q, FAKE, FAKE, None, i64(*shape) if shape else None, i64(*strides) if strides else None, 1.0, out,
                                  None, dtype, ws, wsb, None)


GOOD = (2, 100, 50, 4, 2, 1, 64, 128)


@pytest.mark.parametrize("at,value", [(0, -1), (1, -1), (2, -1), (1, 1 << 30), (2, 1 << 30), (3, 0), (4, 3), (5, 8), (4, 0), (6, 0),
                                      (6, 193), (7, 0), (7, 385), (0, 1 << 24), (3, 1 << 16)])
def test_attention_refuses_shapes(at, value):
    bad = list(GOOD)
    bad[at] = value
    assert fwd(bad) == ERR_ARG
    assert b"attn" in _lib.lib().vx_last_error()
    lib = _lib.lib()
    assert lib.vx_attn_fwd_workspace_bytes(i64(*bad), 0) == 0 and lib.vx_attn_bwd_workspace_bytes(i64(*bad), 0) == 0
    rc = lib.vx_attn_bwd(FAKE, i64(1, 1, 1), FAKE, FAKE, FAKE, None, i64(*bad), i64(*(1,) * 10), FAKE, FAKE, 1.0, FAKE, FAKE, FAKE, 0,
                         FAKE, 1 << 40, None)
    assert rc == ERR_ARG


def test_attention_refuses_arguments():
    lib = _lib.lib()
    assert fwd(None) == ERR_ARG and fwd(GOOD, strides=None) == ERR_ARG
    assert fwd(GOOD, strides=(1,) * 9 + (-1,)) == ERR_ARG
    assert fwd(GOOD, q=None) == ERR_ARG and fwd(GOOD, out=None) == ERR_ARG and fwd(GOOD, dtype=2) == ERR_ARG
    few = (1, 1, 4096, 1, 1, 1, 64, 64)                    # one query: the keys are split, partial sums need room
    need = lib.vx_attn_fwd_workspace_bytes(i64(*few), 0)
    assert need > 0 and fwd(few, wsb=need - 1) == ERR_WS and fwd(few, ws=None, wsb=0) == ERR_WS
    need = lib.vx_attn_bwd_workspace_bytes(i64(*GOOD), 0)
    bwd = lambda ws, n, st: lib.vx_attn_bwd(FAKE, i64(*st), FAKE, FAKE, FAKE, None, i64(*GOOD), i64(*(1,) * 10), FAKE, FAKE, 1.0,  # noqa: E731
                                            FAKE, FAKE, FAKE, 0, ws, n, None)
    assert need > 0 and bwd(FAKE, need - 1, (1, 1, 1)) == ERR_WS and bwd(None, need, (1, 1, 1)) == ERR_WS
    assert bwd(FAKE, need, (1, -1, 1)) == ERR_ARG


def test_attention_workspace_is_bounded():
    """Probabilities and score gradients of any number of queries stay within 256 MiB + what single tiles need."""
    lib = _lib.lib()
    for sq in (1000, 25600, 400000):
        slabs_and_rows = 2 * (-(-sq // 64) + 1) * 1920 * 576 * 4
        assert lib.vx_attn_bwd_workspace_bytes(i64(1, sq, 1920, 2, 2, 1, 192, 384), 0) < (300 << 20) + slabs_and_rows
    for n in (0, 1):                                       # nothing to do: no workspace, no launch
        assert lib.vx_attn_fwd_workspace_bytes(i64(n, 1 - n, 8, 1, 1, 1, 8, 8), 0) in (0, 0)


def test_empty_calls_launch_nothing():
    lib = _lib.lib()
    assert fwd((0, 5, 5, 1, 1, 1, 8, 8)) == 0 and fwd((2, 0, 5, 1, 1, 1, 8, 8)) == 0
    assert lib.vx_linear_fwd(None, 8, None, 8, None, None, 0, 0, 4, 8, 0, None, None, 0, None) == 0


def test_linear_refuses_arguments():
    lib = _lib.lib()
    f = lambda x=FAKE, ldx=8, m=3, n=4, k=8, act=0, dtype=0: lib.vx_linear_fwd(x, ldx, FAKE, 8, None, None, 0, m, n, k, act, FAKE,  # noqa: E731
                                                                              None, dtype, None)
    for kw in (dict(x=None), dict(ldx=-1), dict(m=-1), dict(m=1 << 31), dict(n=0), dict(k=0), dict(n=(1 << 20) + 1), dict(act=4),
               dict(act=-1), dict(dtype=2)):
        assert f(**kw) == ERR_ARG, kw
    need = lib.vx_linear_bwd_workspace_bytes(3, 4, 8, 0)
    b = lambda ws=FAKE, n=need, act=0, saved=None, dpre=None, ld=4: lib.vx_linear_bwd(FAKE, ld, FAKE, 8, FAKE, 8, saved, 3, 4, 8,  # noqa: E731
                                                                                      act, dpre, FAKE, FAKE, FAKE, 0, ws, n, None)
    assert need > 0 and b(n=need - 1) == ERR_WS and b(ws=None) == ERR_WS and b(ld=-1) == ERR_ARG
    assert b(act=1) == ERR_ARG and b(act=1, saved=FAKE) == ERR_ARG and b(act=2, dpre=FAKE) == ERR_ARG


def test_python_refuses_cpu_tensors():
    t = torch.zeros
    with pytest.raises(_lib.VxError):
        fused_tail.attention(t(1, 2, 1, 4), t(1, 2, 1, 4), t(1, 2, 1, 4))
    with pytest.raises(_lib.VxError):
        fused_tail.linear_act(t(2, 3), t(4, 3))
    with pytest.raises(_lib.VxError):
        ops.linear_bwd(t(2, 4), t(2, 3), t(4, 3))
    with pytest.raises(ValueError):
        fused_tail.linear_act(t(2, 5, 3), t(4, 3), None, t(2, 4))


def test_fuse_cross_attention_keeps_keys_and_parameters():
    m = dense_tail.Cross_Attention_Decouple(16, 16, 16, 2, (8, 8), (4, 4), (8, 4), (4, 4), 24)
    sd = {k: v.data_ptr() for k, v in m.state_dict().items()}
    out = fused_tail.fuse_cross_attention(m)
    assert out is m and {k: v.data_ptr() for k, v in m.state_dict().items()} == sd
    kinds = [type(c).__name__ for c in m.modules()]
    assert kinds.count("FusedConvAttention") == 1 and kinds.count("FusedFeedForward") == 2
    fused_tail.fuse_cross_attention(m)                      # again: nothing left to swap
    assert [type(c).__name__ for c in m.modules()] == kinds
    ffn = fused_tail.fuse_cross_attention(dense_tail.FeedFowardLayer(8, 16).eval())
    assert isinstance(ffn, fused_tail.FusedFeedForward) and not ffn.training


def entry_points():
    t = lambda *s: torch.randn(s)  # noqa: E731
    q, k, v, st = t(1, 2, 1, 4), t(1, 2, 1, 4), t(1, 2, 1, 4), t(1, 2, 2)
    x, w, dy = t(2, 3), t(4, 3), t(2, 4)
    return [(fused_tail.attention, (q, k, v)), (ops.attn_fwd, (q, k, v)), (ops.attn_bwd, (q, q, k, v, q, st)),
            (fused_tail.linear_act, (x, w)), (ops.linear_fwd, (x, w)), (ops.linear_bwd, (dy, x, w))]


@pytest.mark.parametrize("at", range(6))
@pytest.mark.parametrize("grad", [False, True])
def test_a_recording_is_refused(at, grad):
    """A trace would keep the allocation of the output and lose the launch: uninitialised memory."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args = entry_points()[at]
    with torch.set_grad_enabled(grad):
        with pytest.raises(_lib.VxError, match="traced"):
            torch.jit.trace(lambda *a: f(*a), args, check_trace=False)
        with pytest.raises(_lib.VxError, match="traced"):
            make_fx(lambda *a: f(*a))(*args)
    with pytest.raises(_lib.VxError, match="CUDA"):          # outside of one: no CPU path, as ever
        f(*args)


@pytest.mark.parametrize("at", range(6))
@pytest.mark.parametrize("arg", [0, 1])
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(at, arg, grad):
    """Forward-mode derivatives: with no input that requires gradients the output came without a tangent."""
    from torch.autograd import forward_ad
    f, args = entry_points()[at]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = list(args)
        dual[arg] = forward_ad.make_dual(args[arg], torch.ones_like(args[arg]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)
        with pytest.raises(_lib.VxError, match="CUDA"):
            f(*args)


def layers():
    torch.manual_seed(0)
    return dense_tail.ConvAttentionLayer_Decouple(16, 2), dense_tail.FeedFowardLayer(16, 24)


DIRECT = [(0, "v_conv"), (0, "out_sem_conv"), (0, "out_geo_conv"), (1, "linear1"), (1, "linear2"), (1, "activation")]


@pytest.mark.parametrize("kind", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                                  "register_full_backward_pre_hook"])
@pytest.mark.parametrize("which,child", DIRECT + [(0, None), (1, None)])
def test_fusing_refuses_hooks(which, child, kind):
    both = torch.nn.ModuleList(layers())
    m = both[which] if child is None else getattr(both[which], child)
    handle = getattr(m, kind)(lambda *a: None)
    with pytest.raises(ValueError, match="hooks"):
        fused_tail.fuse_cross_attention(both)
    assert [type(c) for c in both] == [dense_tail.ConvAttentionLayer_Decouple, dense_tail.FeedFowardLayer]      # nothing changed
    handle.remove()
    both[0].q_sem_conv.register_forward_hook(lambda *a: None)       # called as ever: no reason to refuse
    both[1].norm.register_forward_hook(lambda *a: None)
    fused_tail.fuse_cross_attention(both)
    assert [type(c) for c in both] == [fused_tail.FusedConvAttention, fused_tail.FusedFeedForward]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("which,child", DIRECT[:5])
def test_weights_made_in_a_hook_are_never_stale(which, child):
    """weight_norm makes the weight in a forward pre-hook. Refused when it is there before; when it comes later the layer's own forward
    runs (on the CPU here), with the weight of the present weight_g."""
    x = torch.randn(2, 16, 3, 4) if which == 0 else torch.randn(12, 2, 16)
    call = (lambda m: m(x, x, x, need_maps=False)[0]) if which == 0 else (lambda m: [m(x)])
    stock, plain = layers()[which], layers()[which]
    fused = fused_tail.fuse_cross_attention(layers()[which])
    for m in (stock, fused, plain):
        torch.nn.utils.weight_norm(getattr(m, child))
    with pytest.raises(ValueError, match="hooks"):
        fused_tail.fuse_cross_attention(plain)
    for m in (stock, fused):
        with torch.no_grad():
            getattr(m, child).weight_g.mul_(1.7)
    assert all(torch.equal(a, b) for a, b in zip(call(stock), call(fused)))
    if which == 0:
        with pytest.raises(ValueError, match="key_mask"):
            fused(x, x, x, need_maps=False, key_mask=torch.ones(2, 12, dtype=torch.bool))


def test_fusing_keeps_what_a_layer_holds():
    """Training flags of single submodules, submodules under two names, parameters and buffers of the layer itself, attributes, and a
    layer that stands in two places."""
    att, ffn = layers()
    att.geo_norm = att.sem_norm
    att.out_sem_conv.eval()
    att.register_parameter("gain", torch.nn.Parameter(torch.ones(3)))
    att.register_buffer("seen", torch.zeros(2))
    att.note = "kept"
    net = torch.nn.ModuleList([att, ffn, torch.nn.Sequential(ffn)])
    keys, flags = list(net.state_dict()), {n: m.training for n, m in net.named_modules()}
    ids = {n: id(p) for n, p in net.named_parameters()}
    fused_tail.fuse_cross_attention(net)
    assert type(net[0]) is fused_tail.FusedConvAttention and type(net[1]) is fused_tail.FusedFeedForward
    assert list(net.state_dict()) == keys and {n: m.training for n, m in net.named_modules()} == flags
    assert {n: id(p) for n, p in net.named_parameters()} == ids
    assert net[0].geo_norm is net[0].sem_norm and net[0].note == "kept" and net[1] is net[2][0]
    net[0].extra = torch.nn.Identity()                      # what the replacement gets later is its own
    assert "extra" not in att._modules


def test_layers_that_the_kernels_do_not_compute_are_left_alone():
    """Heads wider than the kernels' (512 channels in one head: 256 / 512; 384 with unreduced keys: 384 / 384), and submodules of another
    kind: the layer stays, or, replaced after the rewriting, runs its own forward."""
    wide = torch.nn.ModuleList([dense_tail.ConvAttentionLayer_Decouple(512, 1), dense_tail.ConvAttentionLayer_Decouple(384, 1, 1),
                                dense_tail.ConvAttentionLayer_Decouple(384, 1), dense_tail.ConvAttentionLayer_Decouple(512, 2)])
    fused_tail.fuse_cross_attention(wide)
    own, fused = dense_tail.ConvAttentionLayer_Decouple, fused_tail.FusedConvAttention
    assert [type(m) for m in wide] == [own, own, fused, fused]

    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return super().forward(x) * 2

    def change(i, m):
        if i < 2:
            m[1].activation = (torch.nn.GELU(), torch.nn.Identity())[i]
        elif i == 2:
            m[1].linear1 = Scaled(16, 24)
        elif i == 3:
            m[1].linear2 = torch.nn.Sequential(torch.nn.Linear(24, 16))
        else:
            name = ("v_conv", "out_geo_conv", "out_sem_conv")[i - 4]
            setattr(m[0], name, torch.nn.Conv2d(16, 16, 3, 1, 1) if i < 6 else torch.nn.Sequential(torch.nn.Conv2d(16, 16, 1)))

    x = torch.randn(2, 16, 3, 4)
    call = lambda m, i: m[0](x, x, x, need_maps=False)[0] if i >= 4 else [m[1](x.flatten(2).permute(2, 0, 1))]  # noqa: E731
    for i in range(7):
        torch.manual_seed(i)
        stock = torch.nn.ModuleList(layers())
        change(i, stock)
        want = call(stock, i)
        before = [type(m) for m in stock]
        fused_tail.fuse_cross_attention(stock)
        kinds = [type(m) for m in stock]
        assert kinds[i < 4] is before[i < 4] and kinds[i >= 4] is not before[i >= 4]
        assert all(torch.equal(a, b) for a, b in zip(call(stock, i), want))
        late = fused_tail.fuse_cross_attention(torch.nn.ModuleList(layers()))
        change(i, late)
        late.load_state_dict(stock.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(call(late, i), want))
    norm = torch.nn.utils.parametrizations.weight_norm
    m = torch.nn.ModuleList(layers())
    norm(m[0].v_conv), norm(m[1].linear1)                    # made at each read of the weight: no hook, never stale
    assert [type(c) for c in fused_tail.fuse_cross_attention(m)] == [fused, fused_tail.FusedFeedForward]


def test_rest_of_the_output():
    """What the forward pass hands to the backward one beside the statistics: bf16 of more than 128 keys alone; refusals as without it."""
    lib = _lib.lib()
    size = lambda dtype, *s: lib.vx_attn_rest_bytes(i64(*s), dtype)  # noqa: E731
    assert size(1, 3, 50, 129, 4, 2, 1, 64, 129) == 3 * 50 * 4 * 129 * 2
    assert size(1, 3, 50, 128, 4, 2, 1, 64, 129) == 0 and size(0, 3, 50, 129, 4, 2, 1, 64, 129) == 0
    assert size(1, 3, 50, 129, 4, 3, 1, 64, 129) == 0 and size(2, 3, 50, 129, 4, 2, 1, 64, 129) == 0
    one = i64(*(1,) * 10)
    assert lib.vx_attn_fwd_rest(FAKE, FAKE, FAKE, None, i64(*GOOD), one, 1.0, None, None, FAKE, 1, FAKE, 1 << 40, None) == ERR_ARG
    assert lib.vx_attn_bwd_rest(FAKE, i64(1, 1, 1), FAKE, FAKE, FAKE, None, i64(*GOOD), one, None, FAKE, FAKE, 1.0, FAKE, FAKE, FAKE, 1,
                                FAKE, 1 << 40, None) == ERR_ARG
    assert lib.vx_attn_bwd_rest(FAKE, i64(1, 1, 1), FAKE, FAKE, FAKE, None, i64(*GOOD), one, FAKE, FAKE, FAKE, 1.0, FAKE, FAKE, FAKE, 1,
                                FAKE, 8, None) == ERR_WS


def test_layer_gradients_workspace_follows_the_activation():
    lib = _lib.lib()
    m, n, k = 1000, 96, 64
    size = [[lib.vx_linear_bwd_act_workspace_bytes(m, n, k, act, dtype) for act in range(4)] for dtype in (0, 1)]
    assert len(set(size[0])) == 1 and size[1][0] == size[1][1] and size[1][2] == size[1][3] == size[1][0] + m * n * 4
    assert [lib.vx_linear_bwd_workspace_bytes(m, n, k, dtype) for dtype in (0, 1)] == [size[0][0], size[1][2]]
    call = lambda act, room: lib.vx_linear_bwd(FAKE, n, FAKE, k, FAKE, k, FAKE, m, n, k, act, FAKE, FAKE, FAKE, FAKE, 1, FAKE, room, None)  # noqa: E731
    assert call(2, size[1][2] - 1) == ERR_WS and call(3, size[1][0]) == ERR_WS and call(1, size[1][1] - 1) == ERR_WS


SHAPES = [(4, 25600, 25600, 2, 2, 1, 192, 384), (8, 25600, 25600, 8, 8, 8, 48, 48), (1, 1024, 57000, 16, 16, 16, 8, 8),
          (1, 25600, 1920, 2, 2, 1, 192, 384), (1, 400000, 1920, 2, 2, 1, 192, 384), (4, 1600, 480, 2, 2, 1, 192, 384),
          (1, 200000, 16, 8, 8, 8, 64, 64), (64, 65, 5001, 8, 4, 2, 40, 60), (1, 3100, 60001, 1, 1, 1, 16, 24), (2, 3000, 129, 16, 16, 16, 32, 32),
          *((4, n, k, 2, 2, 1, 192, 384) for n in (200000, 800000) for k in (200, 2000, 20000))]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_workspace_keeps_its_limits(shape, dtype):
    """Term by term: P and dS of one chunk (1 GiB, or 128 queries of every head where that is more), the slabs of ONE chunk, delta, the
    lists of keys and gathered k and v. Slabs: 2 a CU of at most 128 x 192 tiles in all (512 * 128 * 192 floats), or a split for every
    2 k_len queries of a chunk, rounded up. None of it but delta grows with the number of chunks."""
    b, sq, sk, h, hk, hv, d, dv = shape
    bh, skp, e = b * h, -(-sk // 8) * 8, (4, 2)[dtype]
    chunk = max(1 << 30, 2 * bh * 128 * skp * 4)
    slabs = max(512 * 128 * 192 * 4, bh * (d + dv) * 4 * (min(sq, max(2 ** 29 // (bh * skp * 4), 128)) // 2 + sk))
    rest = bh * sq * 4 + 8 * b * sk + 4 * b + b * sk * (hk * d + hv * dv) * e
    size = _lib.lib().vx_attn_bwd_workspace_bytes(i64(*shape), dtype)
    assert size <= chunk + slabs + rest + 9 * 256
    small = 2 * bh * min(sq, 128) * skp * 4 + bh * sk * (d + dv) * 4 + rest                       # (it is a real amount)
    assert size >= small // 2



def test_no_gradient_wanted_launches_nothing():
    lib = _lib.lib()
    call = lambda dout: lib.vx_attn_bwd(dout, i64(1, 1, 1), FAKE, FAKE, FAKE, None, i64(*GOOD), i64(*(1,) * 10), FAKE, FAKE, 1.0,  # noqa: E731
                                        None, None, None, 0, FAKE, 1 << 40, None)
    assert call(FAKE) == 0 and call(None) == ERR_ARG


def test_launches_past_the_limit_are_refused():
    """One launch has fewer than 2^32 work items: what would need more (and a tensor of that size could be there) is refused by name."""
    lib = _lib.lib()
    rows = (1 << 31) - 1                                   # 2^24 tiles of 128 rows, 256 work items each
    assert lib.vx_linear_fwd(FAKE, 1, FAKE, 1, None, None, 0, rows, 1, 1, 0, FAKE, None, 0, None) == ERR_ARG
    assert b"too many" in lib.vx_last_error()
    assert lib.vx_linear_bwd(FAKE, 1, FAKE, 1, FAKE, 1, None, rows, 1, 1, 0, None, FAKE, None, None, 0, FAKE, 1 << 40, None) == ERR_ARG
    assert b"too many" in lib.vx_last_error()
    many = (1 << 23, 100, 20, 1, 1, 1, 4, 4)
    assert fwd(many) == ERR_ARG and b"too many" in lib.vx_last_error()
    assert lib.vx_attn_bwd(FAKE, i64(1, 1, 1), FAKE, FAKE, FAKE, None, i64(*many), i64(*(1,) * 10), FAKE, FAKE, 1.0, FAKE, FAKE, FAKE, 0,
                           FAKE, 1 << 45, None) == ERR_ARG
    assert b"too many" in lib.vx_last_error()
