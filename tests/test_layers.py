"""Argument checks of the head layers (model/layers.py, include/mdx.h
mdx_linear* / mdx_grouped_linear* / mdx_layer_norm*): every refusal happens on
the host, before any device work, so it is checked without a GPU."""
import ctypes

import pytest
import torch

F32, F16, BF16, I32, I64 = torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int64


@pytest.fixture(scope="module")
def L(mdx):
    from moseq2_detectron_extract_amd.model import layers
    return layers


def z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("err,args,kw", [
    (TypeError, (z(4, 8, dtype=I32), z(3, 8)), {}),                      # x not floating
    (TypeError, (z(4, 8, dtype=torch.float64), z(3, 8)), {}),
    (TypeError, ([[1.0]], z(3, 8)), {}),
    (TypeError, (z(4, 8), z(3, 8, dtype=F16)), {}),                      # weight of another type
    (ValueError, (z(4, 8), z(3, 9)), {}),                                # K differs
    (ValueError, (z(4, 8), z(8)), {}),
    (ValueError, (z(4, 8), z(0, 8)), {}),
    (ValueError, (z(4, 0), z(3, 0)), {}),
    (TypeError, (z(4, 8), z(3, 8), z(3)), {}),                           # bias not float32
    (ValueError, (z(4, 8), z(3, 8), z(4, dtype=F32)), {}),
    (ValueError, (z(4, 8), z(3, 8), None, z(4, 4)), {}),                 # residual's shape
    (TypeError, (z(4, 8), z(3, 8), None, z(4, 3, dtype=F32)), {}),
    (ValueError, (z(4, 8), z(3, 8), None, None, "tanh"), {}),
    (ValueError, (z(4, 8), z(3, 8)), {"out": z(4, 4)}),
    (TypeError, (z(4, 8), z(3, 8)), {"out": z(4, 3, dtype=F32)}),
    (ValueError, (z(4, 8), z(3, 8)), {}),                                # no GPU tensor: no fallback
])
def test_linear_refuses(L, err, args, kw):
    with pytest.raises(err):
        L.linear(*args, **kw)


@pytest.mark.parametrize("err,args,kw", [
    (TypeError, (None, z(4, 8), z(3, 8)), {}),
    (ValueError, (z(4, 4), z(4, 8), z(3, 8)), {}),                       # grad's shape
    (TypeError, (z(4, 3, dtype=F32), z(4, 8), z(3, 8)), {}),
    (ValueError, (z(4, 3), z(4, 8), z(3, 8), None, "relu"), {}),         # activation without pre
    (ValueError, (z(4, 3), z(4, 8), z(3, 8), z(4, 8), "relu"), {}),
    (ValueError, (z(4, 3), z(4, 8), z(3, 8), None, "other"), {}),
    (ValueError, (z(4, 3), z(4, 8), z(3, 8)), {}),                       # on the CPU
])
def test_linear_backward_refuses(L, err, args, kw):
    with pytest.raises(err):
        L.linear_backward(*args, **kw)


@pytest.mark.parametrize("err,args", [
    (ValueError, (z(2, 4, 8), z(2, dtype=I32), z(2, 3, 8))),             # x not (T, K)
    (ValueError, (z(8), z(2, dtype=I32), z(2, 3, 8))),
    (ValueError, (z(4, 8), z(2, dtype=I32), z(3, 8))),                   # weight not (E, N, K)
    (TypeError, (z(4, 8), z(2, dtype=I64), z(2, 3, 8))),                 # counts int32
    (ValueError, (z(4, 8), z(3, dtype=I32), z(2, 3, 8))),                # one count per group
    (ValueError, (z(4, 8), z(4, dtype=I32)[::2], z(2, 3, 8))),           # counts contiguous
    (ValueError, (z(4, 8), z(4097, dtype=I32), z(4097, 1, 8))),          # too many groups
    (ValueError, (z(4, 8), z(2, dtype=I32), z(2, 3, 8), z(3, dtype=F32))),  # bias (E, N)
    (ValueError, (z(4, 8), z(2, dtype=I32), z(2, 3, 8))),                # on the CPU
])
def test_grouped_linear_refuses(L, err, args):
    with pytest.raises(err):
        L.grouped_linear(*args)
    if len(args) == 3:
        with pytest.raises(err):
            L.grouped_linear_backward(z(4, 3), *args)


@pytest.mark.parametrize("err,args,kw", [
    (TypeError, (z(4, 8, dtype=I32),), {}),
    (ValueError, (z(4, 0),), {}),
    (ValueError, (z(()),), {}),
    (TypeError, (z(4, 8), z(8)), {}),                                    # gamma not float32
    (ValueError, (z(4, 8), z(7, dtype=F32)), {}),
    (ValueError, (z(4, 8), None, z(4, 8, dtype=F32)), {}),
    (ValueError, (z(4, 8),), {"eps": -1.0}),
    (ValueError, (z(4, 8),), {"eps": float("nan")}),
    (ValueError, (z(4, 8),), {"out": z(8, 4)}),
    (ValueError, (z(4, 8),), {}),                                        # on the CPU
])
def test_layer_norm_refuses(L, err, args, kw):
    with pytest.raises(err):
        L.layer_norm(*args, **kw)


@pytest.mark.parametrize("err,args", [
    (TypeError, (z(4, 8), z(4, 8), None, z(4, dtype=F32))),
    (ValueError, (z(4, 7), z(4, 8), z(4, dtype=F32), z(4, dtype=F32))),
    (ValueError, (z(4, 8), z(4, 8), z(4, 1, dtype=F32), z(4, dtype=F32))),
    (TypeError, (z(4, 8), z(4, 8), z(4), z(4, dtype=F32))),
    (ValueError, (z(4, 8), z(4, 8), z(4, dtype=F32), z(4, dtype=F32))),  # on the CPU
])
def test_layer_norm_backward_refuses(L, err, args):
    with pytest.raises(err):
        L.layer_norm_backward(*args)


def test_requires_grad_is_refused(L):
    x, w = z(4, 8, dtype=F32), z(3, 8, dtype=F32).requires_grad_()
    with pytest.raises(ValueError, match="requires grad"):
        L.linear(x, w)
    with pytest.raises(ValueError, match="requires grad"):
        L.layer_norm(x.requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):  # past that check
        L.linear(x, w)


def test_rows_and_overlap(L):
    """Which layouts are taken as they are, and which outputs are refused."""
    buf = torch.zeros(6, 40)
    for t, step in ((buf, 40), (buf[:, 3:17], 40), (buf[::2, :5], 80), (buf[:1, :7], 7), (buf.view(2, 3, 40)[:, :, 1:9], 40),
                    (buf.view(2, 3, 40)[:, :1, :9], 120), (buf[:, :1], 40)):
        r = L._rows(t, copy=False)
        assert r.shape == (t.numel() // t.shape[-1], t.shape[-1]) and r.data_ptr() == t.data_ptr()
        assert r.stride(0) == step and torch.equal(r, t.reshape(r.shape))
    for t in (buf.t(), buf[:, ::2], buf[:1].expand(6, 40), buf.view(2, 3, 40)[:, :2]):
        assert L._rows(t, copy=False) is None
        assert L._rows(t).stride() == (t.shape[-1], 1) and torch.equal(L._rows(t), t.reshape(-1, t.shape[-1]))
    a, b = buf[:, :20], buf[:, 20:]
    assert not L._overlap(a, b) and not L._overlap(b, a) and not L._overlap(buf[:3], buf[3:])
    assert L._overlap(a, buf[:, 19:30]) and L._overlap(buf[:4], buf[3:]) and L._overlap(a, a)
    assert not L._overlap(buf[1:, :20], buf[:5, 20:])
    assert L._overlap(torch.as_strided(buf, (3, 10), (60, 1)), a)  # other distances: refused by range
    x = z(0, 8)
    assert L._rows(x).shape == (0, 8) and not L._overlap(x, x)


def _refused(name, *args):
    from moseq2_detectron_extract_amd._lib import lib
    rc = getattr(lib(), name)(*args)
    return rc, lib().mdx_last_error().decode()


def test_c_entry_refusals(mdx):
    """The C entries check before they touch the device: the pointers here
    are never read."""
    p, nul = ctypes.c_void_p(64), None

    def fwd(x=p, ldx=8, w=p, ldw=8, M=4, N=3, K=8, act=0, dtype=3, ldp=0, pre=nul, out=p, ldo=3):
        return _refused("mdx_linear", x, ldx, w, ldw, nul, nul, 0, M, N, K, act, dtype, pre, ldp, out, ldo, nul, 0, nul)
    for kw, msg in (({"dtype": 2}, "dtype"), ({"act": 9}, "activation"), ({"N": 0}, "shape"), ({"M": -1}, "shape"),
                    ({"M": 1 << 31}, "shape"), ({"x": nul}, "null"), ({"out": nul}, "null"), ({"ldx": 7}, "stride"),
                    ({"ldo": 2}, "stride"), ({"pre": p, "ldp": 2}, "stride")):
        rc, text = fwd(**kw)
        assert rc == -1 and msg in text, (kw, rc, text)
    assert fwd(M=0, x=nul, out=nul)[0] == 0  # no rows: nothing to do

    def bwd(grad=p, w=p, pre=nul, act=0, dx=p, dw=nul, db=nul, lddx=8, ws=nul, wsb=0):
        return _refused("mdx_linear_backward", grad, 3, p, 8, w, 8, pre, 3, 4, 3, 8, act, 3, dx, lddx, dw, 8, db, nul, 0,
                        ws, wsb, nul)
    for kw, msg in (({"grad": nul}, "null"), ({"act": 1}, "pre-activation"), ({"w": nul}, "weight"),
                    ({"lddx": 7}, "stride"), ({"db": p}, "workspace"), ({"act": 1, "pre": p}, "workspace"),
                    ({"db": p, "ws": p, "wsb": 1}, "workspace")):
        rc, text = bwd(**kw)
        assert rc == -1 and msg in text, (kw, rc, text)

    def grp(counts=p, E=2, T=4):
        return _refused("mdx_grouped_linear", p, 8, p, nul, nul, 0, counts, E, T, 3, 8, 0, 3, nul, 0, p, 2, 0, nul)
    for kw, msg in (({"counts": nul}, "counts"), ({"E": 0}, "group"), ({"E": 4097}, "groups"), ({}, "stride")):
        rc, text = grp(**kw)
        assert rc == -1 and msg in text, (kw, rc, text)
    assert grp(T=0)[0] == 0

    def nrm(x=p, ldx=8, rows=4, D=8, eps=1e-5, dtype=1, ldo=8):
        return _refused("mdx_layer_norm", x, ldx, nul, nul, rows, D, eps, dtype, p, ldo, nul, nul, nul)
    for kw, msg in (({"x": nul}, "null"), ({"ldx": 7}, "stride"), ({"ldo": 7}, "stride"), ({"D": 0}, "shape"),
                    ({"rows": -1}, "shape"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
                    ({"dtype": 2}, "dtype"), ({"rows": 1 << 22, "D": 1 << 20, "ldx": 1 << 20, "ldo": 1 << 20}, "rows")):
        rc, text = nrm(**kw)
        assert rc == -1 and msg in text, (kw, rc, text)
    assert nrm(rows=0, x=nul)[0] == 0

    def nbk(grad=p, dgamma=p, ws=nul, wsb=0, lddx=8):
        return _refused("mdx_layer_norm_backward", grad, 8, p, 8, p, p, nul, 4, 8, 1, p, lddx, dgamma, nul, ws, wsb, nul)
    for kw, msg in (({"grad": nul}, "null"), ({"lddx": 7}, "stride"), ({}, "workspace"), ({"ws": p, "wsb": 8}, "workspace")):
        rc, text = nbk(**kw)
        assert rc == -1 and msg in text, (kw, rc, text)


def test_workspace_sizes(mdx):
    """Workspace sizes: none for nothing, none where the reduction is not
    split, and room for what the gradients need."""
    from moseq2_detectron_extract_amd._lib import call
    assert call("mdx_linear_workspace_bytes", 0, 8, 8, 0) == 0
    assert call("mdx_linear_workspace_bytes", 1 << 20, 4096, 64, 3) == 0
    n = call("mdx_linear_workspace_bytes", 1000, 1024, 12544, 3)
    assert n % (1000 * 1024 * 4) == 0
    assert call("mdx_linear_backward_workspace_bytes", 100, 30, 50, 0, 3, 1, 0, 0, 0) == 0
    assert call("mdx_linear_backward_workspace_bytes", 100, 30, 50, 1, 3, 1, 1, 0, 0) >= 100 * 30 * 2
    assert call("mdx_linear_backward_workspace_bytes", 100, 30, 50, 1, 3, 1, 0, 0, 1) == 0  # dz goes to dres
    assert call("mdx_grouped_linear_backward_workspace_bytes", 0, 100, 30, 50, 1, 3, 1, 1, 1, 0) == 0
    assert call("mdx_layer_norm_backward_workspace_bytes", 100, 30, 3) >= 2 * 30 * 4


def test_counts_are_needed(L):
    """Without counts a grouped call is refused, a weight of two axes or not."""
    x, dy = z(4, 8), z(4, 3)
    for w in (z(3, 8), z(2, 3, 8)):
        with pytest.raises(TypeError, match="counts"):
            L.grouped_linear(x, None, w)
        with pytest.raises(TypeError, match="counts"):
            L.grouped_linear_backward(dy, x, None, w)


def test_c_entries_refuse_unaligned_workspaces(mdx):
    """Workspaces hold pieces of 16 bytes."""
    p, odd, nul = ctypes.c_void_p(64), ctypes.c_void_p(72), None
    calls = [("mdx_linear", (p, 8, p, 8, nul, nul, 0, 4, 3, 8, 0, 3, nul, 0, p, 3, odd, 1 << 20, nul)),
             ("mdx_linear_backward", (p, 3, p, 8, p, 8, nul, 0, 4, 3, 8, 0, 3, p, 8, nul, 8, p, nul, 0, odd, 1 << 20, nul)),
             ("mdx_grouped_linear_backward", (p, 3, p, 8, p, nul, 0, p, 2, 4, 3, 8, 0, 3, p, 8, nul, p, nul, 0, 1, odd,
                                              1 << 20, nul)),
             ("mdx_layer_norm_backward", (p, 8, p, 8, p, p, nul, 4, 8, 1, p, 8, p, nul, odd, 1 << 20, nul))]
    for name, args in calls:
        rc, text = _refused(name, *args)
        assert rc == -1 and "16-byte aligned" in text, (name, rc, text)


def test_c_entry_refuses_too_many_bias_columns(mdx):
    """More columns of bias over all groups than a launch has threads for."""
    p, nul = ctypes.c_void_p(64), None
    rc, text = _refused("mdx_grouped_linear_backward", p, 1 << 20, p, 1, p, nul, 0, p, 4096, 4, 1 << 20, 1, 0, 3, nul, 1,
                        nul, p, nul, 0, 1, p, 1 << 50, nul)
    assert rc == -1 and "columns of bias" in text, (rc, text)


def every_call(L, x, dtype=F32):
    """Calls of all entries that get x (4, 8) as their first or second tensor, by name."""
    w, c, s = z(3, 8, dtype=dtype), z(2, dtype=I32), z(4, dtype=F32)
    dy = z(4, 3, dtype=dtype)
    return {"linear": lambda: L.linear(x, w), "grouped_linear": lambda: L.grouped_linear(x, c, z(2, 3, 8, dtype=dtype)),
            "linear_backward": lambda: L.linear_backward(dy, x, w),
            "grouped_linear_backward": lambda: L.grouped_linear_backward(dy, x, c, z(2, 3, 8, dtype=dtype)),
            "layer_norm": lambda: L.layer_norm(x), "layer_norm_backward": lambda: L.layer_norm_backward(z(4, 8, dtype=dtype), x, s, s)}


def test_tangents_are_refused(L):
    """A forward-mode tangent would be lost; requires_grad does not show it."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        x = forward_ad.make_dual(z(4, 8, dtype=F32), torch.ones(4, 8))
        for name, f in every_call(L, x).items():
            with pytest.raises(ValueError, match="tangent"):
                f()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # which leaves tangents alone
                f()
        b = forward_ad.make_dual(z(3, dtype=F32), torch.ones(3))
        with pytest.raises(ValueError, match="tangent"):
            L.linear(z(4, 8, dtype=F32), z(3, 8, dtype=F32), b)
        for f in every_call(L, z(4, 8, dtype=F32)).values():  # a level without tangents is no matter
            with pytest.raises(ValueError, match="GPU"):
                f()
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda a: L.layer_norm(a), (z(4, 8, dtype=F32),), (torch.ones(4, 8),))


@pytest.mark.filterwarnings("ignore")
def test_tracers_are_refused(L):
    """A trace would hold the allocation of the outputs and not the call."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for name in every_call(L, z(4, 8, dtype=F32)):
        f = lambda a: every_call(L, a)[name]()  # noqa: B023, E731
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (z(4, 8, dtype=F32),))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(z(4, 8, dtype=F32))


def test_negative_views(L):
    """The imaginary part of a conjugate is a view that stands for -1 times its memory."""
    for shape in ((1, 1), (5, 1), (3, 4)):
        c = torch.arange(1, 1 + 2 * shape[0] * shape[1], dtype=F32).view(*shape, 2)
        t = torch.view_as_complex(c).conj().imag
        want = -c[..., 1]
        assert t.is_neg()
        for r in (L._rows(t), L._laid(t)[0], L._dense(t)):
            assert not r.is_neg() and r.is_contiguous() and torch.equal(r.view(shape), want)
        assert L._laid(t)[1] == shape[1] and L._rows(t, copy=False) is None
    t = torch._neg_view(torch.ones(3, 4))  # contiguous
    assert torch.equal(L._laid(t)[0], -torch.ones(3, 4)) and not L._laid(t)[0].is_neg() and not L._dense(t).is_neg()


def test_plan(mdx):
    """The kernel of a call: known to the caller, never one whose launch has 2^32 threads, and with slices that the
    workspace has room for."""
    from moseq2_detectron_extract_amd._lib import call
    side, threads = (256, 128, 64, 128, 64), (512, 256, 256, 256, 256)
    for M, N, K in ((1, 1, 1), (33, 8, 16), (1000, 1024, 12544), (2048, 2048, 2048), (6 * 10 ** 8, 8, 16),
                    (12 * 10 ** 8, 8, 16), (2 ** 31 - 65537, 64, 1), (1, 54 * 10 ** 7, 8), (32, 2 ** 31 - 65537, 1)):
        for dtype in (0, 1, 3):
            room = call("mdx_linear_workspace_bytes", M, N, K, dtype)
            for aligned in (0, 1):
                kernel, slices = (lambda p: (p % 16, p // 16))(call("mdx_linear_plan", 0, M, N, K, dtype, aligned, 0))
                assert kernel in ((5, 0, 1, 2) if aligned else (5, 3, 4)) and (kernel or dtype)
                assert slices == 1 or slices * M * N * 4 <= room
                if kernel < 5:
                    tiles = -(-M // side[kernel]) * -(-N // side[kernel]) * slices
                    assert tiles * threads[kernel] < 2 ** 32, (M, N, K, dtype, aligned, kernel)
    assert call("mdx_linear_plan", 0, 4, 1024, 1024, 3, 1, 0) % 16 == 5
    assert call("mdx_linear_plan", 0, 8192, 4096, 1024, 3, 1, 1) % 16 == 0
    assert call("mdx_linear_plan", 8, 64, 4096, 1024, 0, 1, 0) % 16 == 5
    for args in ((0, 4, 0, 8, 3, 1, 0), (4097, 4, 8, 8, 3, 1, 0), (0, 4, 8, 8, 2, 1, 0), (0, -1, 8, 8, 3, 1, 0)):
        assert _refused("mdx_linear_plan", *args)[0] == -1


def test_layer_norm_refuses_many_wide_rows(L):
    """A workgroup for each row of more than 16384 elements: 2^22 of them are refused (an expanded tensor: no memory)."""
    x, s = z(1, 1, dtype=F32).expand(1 << 22, 16385), z(1, dtype=F32).expand(1 << 22)
    with pytest.raises(ValueError, match="rows of more than 16384"):
        L.layer_norm(x)
    with pytest.raises(ValueError, match="rows of more than 16384"):
        L.layer_norm_backward(x, x, s, s)
    with pytest.raises(ValueError, match="GPU"):
        L.layer_norm(x[1:])
    with pytest.raises(ValueError, match="GPU"):
        L.layer_norm(z(1, 1, dtype=F32).expand(1 << 22, 16384))


def test_layers_are_exported(L):
    """The layers are reached from the model package, as the runtime and the predictor are."""
    from moseq2_detectron_extract_amd import model
    for name in ("linear", "linear_backward", "grouped_linear", "grouped_linear_backward", "layer_norm", "layer_norm_backward"):
        assert getattr(model, name) is getattr(L, name)
    from moseq2_detectron_extract_amd.model import layer_norm, linear  # noqa: F401
    with pytest.raises(AttributeError):
        model.other
