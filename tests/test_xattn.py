"""Cross attention and the query / key norm with rotation: what they refuse,
checked without a GPU (every refusal comes before the device check), the C
entries' argument checks, and the rotation's step table."""
import ctypes
from decimal import Decimal, getcontext

import pytest
import torch

from text_guided_face_recognition_amd import _hip
from text_guided_face_recognition_amd import kernels as K


def qkv(b=2, tq=5, tk=7, h=4, hk=2, d=16, dtype=torch.float32):
    return (torch.zeros(b, tq, h, d, dtype=dtype), torch.zeros(b, tk, hk, d, dtype=dtype),
            torch.zeros(b, tk, hk, d, dtype=dtype))


@pytest.mark.parametrize("change,error", [
    (lambda q, k, v: dict(q=q[0]), ValueError),                           # no batch
    (lambda q, k, v: dict(v=v[:, :6]), ValueError),                       # k, v differ
    (lambda q, k, v: dict(q=q.bfloat16()), TypeError),                    # mixed types
    (lambda q, k, v: dict(q=q.double(), k=k.double(), v=v.double()), TypeError),
    (lambda q, k, v: dict(q=q[:1]), ValueError),                          # batches differ
    (lambda q, k, v: dict(q=q[..., :8]), ValueError),                     # head sizes differ
    (lambda q, k, v: dict(q=q[:, :, :3]), ValueError),                    # 3 heads on 2
    (lambda q, k, v: dict(zip("qkv", qkv(d=257))), ValueError),
    (lambda q, k, v: dict(scale=0.0), ValueError),
    (lambda q, k, v: dict(scale=-1.0), ValueError),
    (lambda q, k, v: dict(scale=float("nan")), ValueError),
    (lambda q, k, v: dict(kv_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (lambda q, k, v: dict(kv_lens=torch.zeros(2)), ValueError),
    (lambda q, k, v: dict(q_lens=[1, 2]), ValueError),
    (lambda q, k, v: dict(mask=torch.ones(2, 7)), ValueError),            # not bool
    (lambda q, k, v: dict(mask=torch.ones(2, 5, dtype=torch.bool)), ValueError),
    (lambda q, k, v: dict(), RuntimeError),                               # CPU tensors
])
def test_cross_attention_refuses(change, error):
    q, k, v = qkv()
    with pytest.raises(error):
        K.cross_attention(**{**dict(q=q, k=k, v=v), **change(q, k, v)})


def test_cross_attention_refuses_too_many_rows():
    x = torch.zeros(1, 1, 1, 1).expand(1, (1 << 30) + 1, 1, 1)
    with pytest.raises(ValueError):
        K.cross_attention(x, torch.zeros(1, 1, 1, 1), torch.zeros(1, 1, 1, 1))


def test_cross_attention_refuses_too_many_key_heads():
    """A launch has at most 2^32 - 1 threads, and a key head 256 or more."""
    x = torch.zeros(1, 1, 1, 1).expand(1 << 24, 1, 1, 1)
    with pytest.raises(ValueError):
        K.cross_attention(x, x, x)
    n = ctypes.c_longlong(0)
    for b, ok in ((1 << 24, 1001), ((1 << 24) - 1, 0)):
        for backward in (0, 1):
            assert _hip.lib().tgfr_cross_attention_ws(b, 1, 1, 1, 1, 64, 0, backward,
                                                      ctypes.byref(n)) == ok


def norm_args(d=16, dtype=torch.float32):
    return dict(q=torch.zeros(2, 5, 4, d, dtype=dtype), k=torch.zeros(2, 7, 2, d, dtype=dtype),
                q_weight=torch.ones(d), k_weight=torch.ones(d),
                rope=K.Rope(d, device="cpu") if d % 2 == 0 else None)


@pytest.mark.parametrize("change,error", [
    (dict(q=None, k=None), ValueError),
    (dict(q=torch.zeros(5, 4, 16)), ValueError),
    (dict(q=torch.zeros(2, 5, 4, 16).long()), TypeError),
    (dict(q=torch.zeros(2, 5, 4, 16).bfloat16()), ValueError),            # types differ
    (dict(q_weight=None), ValueError),
    (dict(k_weight=torch.ones(16).bfloat16()), ValueError),
    (dict(k_weight=torch.ones(8)), ValueError),
    (dict(rope=K.Rope(18, device="cpu")), ValueError),                    # more than the head
    (dict(rope=None, q_pos=torch.arange(5)), ValueError),                 # positions of nothing
    (dict(q_pos=torch.arange(5).float()), TypeError),
    (dict(q_pos=torch.arange(4)), ValueError),
    (dict(q_pos=torch.zeros(5, 2).long()), ValueError),
    (dict(rope=K.Rope(16, axes=2, device="cpu")), ValueError),            # axes need positions
    (dict(q_pos=torch.arange(5), k_pos=torch.arange(7).int()), TypeError),
    (dict(eps=-1.0), ValueError),
    (dict(out_dtype=torch.float64), TypeError),
    (dict(), RuntimeError),                                               # CPU tensors
])
def test_qk_norm_rope_refuses(change, error):
    with pytest.raises(error):
        K.qk_norm_rope(**{**norm_args(), **change})


@pytest.mark.parametrize("d", [15, 258])
def test_qk_norm_rope_refuses_head_sizes(d):
    with pytest.raises(ValueError):
        K.qk_norm_rope(**norm_args(d))


def test_qk_norm_rope_refuses_widening():
    with pytest.raises(TypeError):
        K.qk_norm_rope(**norm_args(dtype=torch.bfloat16), out_dtype=torch.float32)


def test_qk_norm_rope_refuses_a_changed_rope():
    """Sizes that a Rope's steps do not fit are refused, never read past."""
    for name, value in (("dim", 12), ("dim", 10), ("axes", 3), ("turn", torch.zeros(8)),
                        ("turn", torch.zeros(16).long()[::2])):
        rope = K.Rope(16, device="cpu")
        setattr(rope, name, value)
        pos = dict(q_pos=torch.zeros(5, 3).long(), k_pos=torch.zeros(7, 3).long()) \
            if rope.axes == 3 else {}
        with pytest.raises(ValueError):
            K.qk_norm_rope(**{**norm_args(), "rope": rope, **pos})


def test_qk_norm_rope_refuses_too_many_tokens():
    """Token numbers are 32-bit."""
    x = torch.zeros(1, 1, 1, 16).expand(1, (1 << 30) + 1, 1, 16)
    with pytest.raises(ValueError):
        K.qk_norm_rope(x, None, torch.ones(16), None)


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_cross_attention_refuses_tangents(which):
    """Forward mode: no derivative is given, and none is dropped in silence."""
    x = dict(zip("qkv", qkv()))
    with torch.autograd.forward_ad.dual_level():
        x[which] = torch.autograd.forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            K.cross_attention(**x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            K.cross_attention(**x)


@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight"])
def test_qk_norm_rope_refuses_tangents(which):
    x = norm_args()
    with torch.autograd.forward_ad.dual_level():
        x[which] = torch.autograd.forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            K.qk_norm_rope(**x)


def test_tracing_is_refused():
    """A trace would hold the output's allocation and not the kernel."""
    n = norm_args()
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda *x: K.cross_attention(*x), qkv())
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda q, w: K.qk_norm_rope(q, None, w, None)[0], (n["q"], n["q_weight"]))


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=15), dict(dim=6, axes=2),
                                dict(dim=8, axes=0), dict(dim=8, base=0.5),
                                dict(dim=8, base=float("inf"))])
def test_rope_refuses(kw):
    with pytest.raises(ValueError):
        K.Rope(**kw, device="cpu")


def test_rope_steps():
    """turn[i] = base^(-i / n) / 2 pi of a circle, rounded to 2^-64, the same
    for every axis; pi from Machin's formula."""
    getcontext().prec = 50

    def arctan_inverse(x):
        total, term, n = Decimal(0), Decimal(1) / x, 0
        while abs(term) > Decimal(10) ** -48:
            total += (-1) ** n * term / (2 * n + 1)
            term /= x * x
            n += 1
        return total
    pi = 4 * (4 * arctan_inverse(5) - arctan_inverse(239))
    r = K.Rope(24, base=500.0, axes=2, device="cpu")
    assert r.turn.shape == (12,) and torch.equal(r.turn[:6], r.turn[6:])
    for i in range(6):
        want = (Decimal(500).ln() * -i / 6).exp() / (2 * pi) * 2 ** 64
        assert abs(int(r.turn[i]) - want) <= 1


def test_grid_positions():
    p = K.grid_positions(3, 5, device="cpu")
    assert p.shape == (15, 2)
    assert p.tolist() == [[i, j] for i in range(3) for j in range(5)]


def test_c_entries_check_arguments():
    """Each call returns before any launch."""
    lib = _hip.lib()
    n = ctypes.c_longlong(0)
    ref = ctypes.byref(n)
    ok = dict(B=2, Tq=5, Tk=7, H=4, Hk=2, D=64, type=0)

    def ws(**kw):
        return lib.tgfr_cross_attention_ws(*{**ok, **kw}.values(), 0, ref)
    assert ws() == 0
    for bad in (dict(B=0), dict(Tq=0), dict(Tk=0), dict(H=3), dict(Hk=0), dict(D=0), dict(D=257),
                dict(Tk=(1 << 30) + 1), dict(B=1 << 20, Tk=1 << 12)):
        assert ws(**bad) == 1001, bad
    assert ws(type=3) == 1002
    # a token against long states is split, and the parts need room
    assert ws(B=1, Tq=1, Tk=8192) == 0 and n.value > 0
    # a large batch is not
    assert ws(B=512, Tq=128) == 0 and n.value == 0
    # null pointers; a scale that is not positive
    some = ctypes.addressof(n)
    head = [some, some, some, some, some, None, None, None, 0, 512, 128, 7, 4, 2, 64]
    assert lib.tgfr_cross_attention_fwd(*head, 0.0, 0, None, None, None) == 1001
    assert lib.tgfr_cross_attention_fwd(None, *head[1:], 1.0, 0, None, None, None) == 1001
    # dk without dv; no statistics
    args = [some] * 9 + [None, None, None, 0, 2, 5, 7, 4, 2, 64, 1.0, 0, some, some, None]
    args[7] = None
    assert lib.tgfr_cross_attention_bwd(*args) == 1001
    args[7], args[21] = some, None
    assert lib.tgfr_cross_attention_bwd(*args) == 1001
    assert lib.tgfr_qk_norm_rope_ws(64, ref) == 0 and n.value > 0
    assert lib.tgfr_qk_norm_rope_ws(0, ref) == 1001
    shapes = (ctypes.c_longlong * 30)(2, 5, 4, *[0] * 12, 2, 7, 2, *[0] * 12)
    norm = [some, some, some, some, ctypes.addressof(shapes), some, some, None, None, 0, some, 16,
            1, 0, 16, 1e-6, 0, 0, None]

    def fwd(at, value):
        return lib.tgfr_qk_norm_rope_fwd(*norm[:at], value, *norm[at + 1:])
    for at, value in ((2, None), (4, None), (5, None), (11, 18), (11, 15), (12, 3), (14, 15),
                      (14, 258), (10, None)):
        assert fwd(at, value) == 1001, (at, value)
    assert fwd(16, 3) == 1002 and fwd(17, 1) == 1002      # bf16 is not written as fp32


def test_module_refuses():
    from text_guided_face_recognition_amd.models.fusion_nets import CrossAttention
    for kw in (dict(channel_dim=30, heads=4), dict(channel_dim=32, heads=4, kv_heads=3)):
        with pytest.raises(ValueError):
            CrossAttention(**kw)
