"""Norm + rotation of q and k, linear attention with a decay per head, and its single-token form (include/a2v.h) against plain
recurrences in 64 bits.

Tolerances, per element: |y - y64| <= u |y64| + c A, where u is the half step of the result's type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32),
A is the sum of the magnitudes of the terms that make up y (the same formula on the inputs' absolute values) and c covers what happens
before the one rounding:
  bf16 linear attention   an operand split into hi + lo is off by 2^-8 2^-8 = 2^-16 of itself; a term passes two splits (scaled value,
                          then state; or score) and at most a few hundred fp32 additions (512 x 2^-24 = 2^-15): c = 2^-14
  fp32 linear attention   rows + HD fp32 additions and a handful of products and powers: c = (rows + HD + 64) 2^-24
  norm and rotation       sum of HD squares (HD 2^-24, halved by the root), root and products (8 x 2^-24), sine and cosine (2^-22):
                          c = 2^-18 for HD <= 128
"""
import contextlib
import threading

import pytest
import torch

gpu = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def check(got, want, mag, c, what=""):
    u = U[got.dtype]
    g, w, m = got.detach().double().cpu(), want.double(), mag.double()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    off = (g - w).abs() - (u * w.abs() + c * m)
    assert torch.isfinite(g).all() and float(off.max() if off.numel() else -1.0) <= 0.0, \
        (what, float(off.max()), float((g - w).abs().max()), int((off > 0).sum()), off.numel())


def rnd(*shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ references
def ref_norm_rope(x, w, ang, interleaved, eps, dy=None):
    """x (..., HD) double, ang (..., half); -> y, or dx and the terms of dw"""
    hd, half = x.shape[-1], ang.shape[-1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()

    def turn(z, s):
        out = z.clone()
        out[..., a] = z[..., a] * ang.cos() - s * z[..., b] * ang.sin()
        out[..., b] = z[..., b] * ang.cos() + s * z[..., a] * ang.sin()
        return out
    if dy is None:
        return turn(x * r * w, 1.0)
    g = turn(dy, -1.0)
    gw = g * w
    dx = r * (gw - x * r * (gw * x * r).mean(-1, keepdim=True))
    return dx, g * x * r


def ref_linear(q, k, v, slopes, scale, state=None, d_out=None, d_state=None):
    """one sequence: q (S,H,D), k, v (S,HK,D) double -> out, last [, dq, dk, dv, d_first]"""
    S, H, D = q.shape
    rep = H // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    lam = torch.exp(-slopes.double())[:, None, None]
    st = state.clone() if state is not None else torch.zeros(H, D, D, dtype=torch.float64)
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    for t in range(S):
        st = lam * st + k[t].unsqueeze(-1) * v[t].unsqueeze(-2)
        out[t] = scale * (q[t].unsqueeze(-2) @ st).squeeze(-2)
        if d_out is not None:
            dq[t] = scale * (st @ d_out[t].unsqueeze(-1)).squeeze(-1)
    if d_out is None:
        return out, st
    g = d_state.clone() if d_state is not None else torch.zeros(H, D, D, dtype=torch.float64)
    dk, dv = torch.zeros_like(q), torch.zeros_like(q)
    for t in reversed(range(S)):
        g = g + scale * q[t].unsqueeze(-1) * d_out[t].unsqueeze(-2)
        dk[t] = (g @ v[t].unsqueeze(-1)).squeeze(-1)
        dv[t] = (k[t].unsqueeze(-2) @ g).squeeze(-2)
        g = lam * g
    fold = lambda x: x.reshape(S, H // rep, rep, D).sum(2)      # noqa: E731
    return out, st, dq, fold(dk), fold(dv), g


def c_of(dtype, rows, hd):
    return 2.0 ** -14 if dtype == torch.bfloat16 else (rows + hd + 64) * 2.0 ** -24


def alibi(H, low=0.0):
    return torch.exp2(-8.0 * torch.arange(1, H + 1).float() / H) + low


def test_reference_gradients_are_the_formulas():
    """the references' backward against torch.autograd in 64 bits"""
    S, H, HK, D = 7, 4, 2, 8
    q, k, v = (rnd(S, h, D, seed=i).double().requires_grad_() for i, h in enumerate((H, HK, HK)))
    st = rnd(H, D, D, seed=4).double().requires_grad_()
    do, ds = rnd(S, H, D, seed=5).double(), rnd(H, D, D, seed=6).double()
    slopes = alibi(H)
    lam = torch.exp(-slopes.double())[:, None, None]
    s, outs = st, []
    for t in range(S):
        s = lam * s + k[t].repeat_interleave(2, 0).unsqueeze(-1) * v[t].repeat_interleave(2, 0).unsqueeze(-2)
        outs.append(0.3 * (q[t].unsqueeze(-2) @ s).squeeze(-2))
    (torch.stack(outs) * do).sum().add((s * ds).sum()).backward()
    got = ref_linear(q.detach(), k.detach(), v.detach(), slopes, 0.3, st.detach(), do, ds)
    for a, b in zip(got[2:], (q.grad, k.grad, v.grad, st.grad)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    x, w = rnd(5, 3, 16, seed=1).double().requires_grad_(), rnd(16, seed=2).double().requires_grad_()
    ang, dy = rnd(5, 1, 4, seed=3).double(), rnd(5, 3, 16, seed=4).double()
    for inter in (False, True):
        x.grad = w.grad = None
        i = torch.arange(4)
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + 4)
        y = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        za, zb = y[..., a] * ang.cos() - y[..., b] * ang.sin(), y[..., b] * ang.cos() + y[..., a] * ang.sin()
        (za * dy[..., a] + zb * dy[..., b]).sum().add((y[..., 8:] * dy[..., 8:]).sum()).backward()
        dx, dw = ref_norm_rope(x.detach(), w.detach(), ang, inter, 1e-6, dy)
        assert torch.allclose(dx, x.grad, rtol=1e-12, atol=1e-12) and torch.allclose(dw.sum((0, 1)), w.grad, rtol=1e-12, atol=1e-12)


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def _rope_args(N=2, S=5, H=4, HK=2, HD=64, dtype=torch.bfloat16):
    z = lambda *s, d=dtype: torch.zeros(*s, dtype=d)          # noqa: E731
    return dict(q=z(N, S, H, HD), k=z(N, S, HK, HD), q_weight=z(HD, d=torch.float32), k_weight=z(HD, d=torch.float32), inv_freq=z(HD // 2, d=torch.float32),
                pos=torch.zeros(N, S, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 5, 4, 48, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 5, 256, dtype=torch.bfloat16)),
    dict(k=torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16)), dict(q_weight=torch.zeros(32)), dict(k_weight=torch.zeros(64, dtype=torch.bfloat16)),
    dict(inv_freq=torch.zeros(4)), dict(inv_freq=torch.zeros(33)), dict(inv_freq=torch.zeros(40)), dict(sections=(16, 8)), dict(sections=(8, 8, 8, 8)),
    dict(sections=(40, -8)), dict(pos=None, sections=(16, 16)), dict(pos=torch.zeros(2, 5)), dict(pos=torch.zeros(2, 5, 2, dtype=torch.int32)),
    dict(pos=torch.zeros(5, dtype=torch.int32)), dict(q_out=torch.zeros(2, 5, 4, 64)), dict(q_out=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 5, 64, 4, dtype=torch.bfloat16).transpose(2, 3)), dict(q=torch.zeros(2 * 5 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 5, 4, 64)),
    dict(q_out=torch.zeros(1, 5, 4, 64, dtype=torch.bfloat16).expand(2, 5, 4, 64)), dict(k=torch.zeros(2, 5, 2, 64)),
], ids=lambda c: "-".join(c))
def test_norm_rope_refusals(change):
    from animal2vec_amd import ops
    with pytest.raises((ValueError, TypeError)):
        ops.qk_norm_rope_fwd(**{**_rope_args(), **change})


def test_overlap_of_a_layout_seen_before():
    """a layout's verdict holds for the relative positions it was found at, not for others"""
    from animal2vec_amd import ops
    buf = torch.zeros(4096, dtype=torch.bfloat16)
    t = lambda at: buf.as_strided((1, 4, 2, 64), (512, 128, 64, 1), at)        # noqa: E731
    a, b, far, onto = t(0), t(512), t(2048), t(64)
    rows = buf.view(1, 8, 8, 64)
    spans = ops._spans((a, b), (a, b))
    for _ in range(2):
        ops._apart_again("x", spans, (a, b), (a, b), inplace=True)
        ops._apart_again("x", spans, (a, b), (far, t(2560)), inplace=True)
        for bad in (((a, b), (b, a)), ((a, onto), (a, b)), ((a, b), (far, onto)), ((a, a), (far, b))):
            with pytest.raises(ValueError, match="overlap"):
                ops._apart_again("x", spans, *bad, inplace=True)
    # slots of one packed buffer meet in their ranges and are apart; moved by a head they are not
    q, k, v, o = (rows[:, :, i:i + 2] for i in (0, 2, 4, 6))
    spans = ops._spans((o,), (q, k, v))
    for _ in range(2):
        ops._apart_again("x", spans, (o,), (q, k, v))
        ops._apart_again("x", spans, (q,), (k, v, o))
        with pytest.raises(ValueError, match="overlap"):
            ops._apart_again("x", spans, (rows[:, :, 5:7],), (q, k, v))


def test_outputs_may_not_overlap():
    from animal2vec_amd import ops
    qkv = torch.zeros(2, 5, 3, 4, 64, dtype=torch.bfloat16)
    q, k, v = qkv.unbind(2)
    a = _rope_args()
    rope = dict(a, q=q, k=k)
    for bad in (dict(q_out=k), dict(q_out=v, k_out=v), dict(q_out=q, k_out=q), dict(k_out=q)):
        with pytest.raises(ValueError, match="overlap"):
            ops.qk_norm_rope_fwd(**rope, **bad)
    slopes = torch.zeros(4)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_attention_fwd(q, k, v, slopes, out=q)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_attention_bwd(q, k, v, slopes, torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16), dq=q, dk=k, dv=v)
    d = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_attention_bwd(q, k, v, slopes, torch.zeros_like(d), dq=d, dk=d, dv=torch.zeros_like(d))
    assert not ops._overlap(q, k) and not ops._overlap(v, q) and ops._overlap(q, qkv.view(2, 5, 12, 64)[:, :, 2:6])
    assert not ops._overlap(qkv[0:1, 0:1, 0], qkv[0:1, 0:1, 1]) and ops._overlap(qkv[0:1, 0:1, 0], qkv[0:1, 0:1, 0])
    # packed slots pass these checks and reach the device check
    from animal2vec_amd import _lib
    for go in (lambda: ops.qk_norm_rope_fwd(**rope, q_out=q, k_out=k), lambda: ops.linear_attention_fwd(q, k, v, slopes, out=torch.zeros_like(d))):
        with pytest.raises(_lib.A2VError):
            go()
    w = torch.zeros(96)
    for dk_weight in (w[:64], w[32:]):
        with pytest.raises(ValueError, match="two buffers"):
            ops.qk_norm_rope_bwd(d, d, **dict(a, q=d, k=d), dq_weight=w[:64], dk_weight=dk_weight)
    # one tensor given twice: in place for q would change k under its reader
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_rope_fwd(**dict(a, q=q, k=q), q_out=q)
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_rope_bwd(d, d, **dict(a, q=q, k=k), dq_weight=w[:64], dk_weight=torch.zeros(64), dq=d)
    # rows and heads of an output that meet
    for strides in ((1280, 64, 64, 1), (1280, 128, 64, 1), (256, 256, 64, 1)):
        with pytest.raises(ValueError, match="repeat"):
            ops.linear_attention_fwd(d, d, d, slopes, out=torch.zeros(2 * 1280 * 4, dtype=torch.bfloat16).as_strided((2, 5, 4, 64), strides))


def _lin_args(N=2, S=5, H=4, HK=2, HD=64, dtype=torch.bfloat16):
    return dict(q=torch.zeros(N, S, H, HD, dtype=dtype), k=torch.zeros(N, S, HK, HD, dtype=dtype), v=torch.zeros(N, S, HK, HD, dtype=dtype), slopes=torch.zeros(H))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 5, 3, 64, dtype=torch.bfloat16), slopes=torch.zeros(3)), dict(v=torch.zeros(2, 5, 1, 64, dtype=torch.bfloat16)), dict(slopes=torch.zeros(2)),
    dict(slopes=torch.zeros(4).double()), dict(state=torch.zeros(2, 4, 64, 64, dtype=torch.bfloat16)), dict(state=torch.zeros(1, 4, 64, 64)),
    dict(state=torch.zeros(2, 4, 64, 64).transpose(2, 3)), dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), dict(k=torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16)),
    dict(out=torch.zeros(2, 5, 4, 64)), dict(q=torch.zeros(2, 5, 4, 16, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 5, 4, 64, dtype=torch.float64)),
    dict(q=torch.zeros(2, 5, 4, 64)),
], ids=lambda c: "-".join(c))
def test_linear_attention_refusals(change):
    from animal2vec_amd import ops
    with pytest.raises((ValueError, TypeError)):
        ops.linear_attention_fwd(**{**_lin_args(), **change})


def test_linear_attention_more_refusals():
    from animal2vec_amd import ops
    packed = _lin_args(N=1)
    for cu in (torch.zeros(3, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.linear_attention_fwd(**packed, cu_seqlens=cu)
    a = _lin_args()
    do = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16)
    for bad in (dict(d_out=do[:, :4]), dict(d_out=do, dq=do.clone()), dict(d_out=do, d_state=torch.zeros(2, 4, 64, 32))):
        with pytest.raises((ValueError, TypeError)):
            ops.linear_attention_bwd(**a, **bad)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)      # noqa: E731
    step = dict(q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), slopes=torch.zeros(4), state=torch.zeros(3, 4, 64, 64))
    for bad in (dict(state=torch.zeros(2, 4, 64, 64)), dict(state=z(3, 4, 64, 64)), dict(slots=torch.zeros(3, dtype=torch.int64)), dict(slots=torch.zeros(2, dtype=torch.int32)),
                dict(k=z(2, 2, 64)), dict(q=z(3, 1, 4, 64)), dict(out=z(3, 2, 64)), dict(out=step["q"])):
        with pytest.raises((ValueError, TypeError)):
            ops.linear_attention_step(**{**step, **bad})
    with ops.half_library():
        h = {n: t.half() if t.dtype == torch.bfloat16 else t for n, t in _lin_args().items()}
        with pytest.raises(TypeError, match="float16"):
            ops.linear_attention_fwd(**h)


def test_c_entries_refuse_bad_arguments():
    """argument checks of the C entries: they return before anything is launched (no GPU here)"""
    import ctypes as C
    from animal2vec_amd import _lib
    for lib, half in ((_lib.load(), False), (_lib.load_f16(), True)):
        buf = (C.c_char * 4096)()
        p = (C.addressof(buf) + 63) // 64 * 64
        st = (C.c_longlong * 21)(*([64] * 21))
        sec = (C.c_int * 3)(16, 8, 8)

        def fwd(dtype=0, q=p, k=p, v=p, o=p, st=st, sl=p, B=1, S=4, H=2, HK=2, HD=64, ws=None, n=0):
            return lib.a2v_linear_attention_fwd(dtype, q, k, v, o, st, sl, None, None, None, B, S, H, HK, HD, 1.0, 0, ws, n, None)
        assert fwd(dtype=7) == -2 and fwd(q=None) == -1 and fwd(o=p + 4) == -1 and fwd(st=None) == -1 and fwd(sl=None) == -1 and fwd(H=3) == -1 and fwd(HD=48) == -1
        assert fwd(st=(C.c_longlong * 12)(*([66] * 12))) == -1 and fwd(B=0) == 0 and fwd(B=-1) == -1 and fwd(S=1 << 30) == -1
        assert fwd(B=1, S=100000) == -1                            # no workspace
        assert fwd(B=1, S=1, H=1 << 16, HK=1 << 16) == -1          # 2^28 elements of state in one sequence
        # a state that is left where one is read
        n = 2 * 64 * 64 * 4
        for first, last in ((p, p), (p, p + n - 16), (p + n - 16, p)):
            assert lib.a2v_linear_attention_fwd(0, p, p, p, p, st, p, first, last, None, 1, 4, 2, 2, 64, 1.0, 0, None, 0, None) == -1
            assert lib.a2v_linear_attention_bwd(0, p, p, p, p, p, p, p, st, p, first, None, last, None, 1, 4, 2, 2, 64, 1.0, 0, None, 0, None) == -1
            assert lib.a2v_linear_attention_bwd(0, p, p, p, p, p, p, p, st, p, None, first, last, None, 1, 4, 2, 2, 64, 1.0, 0, None, 0, None) == -1
        assert fwd(dtype=1, B=0) == (-4 if half else 0)
        need = lib.a2v_linear_attention_workspace(0, 1, 0, 1, 100000, 2, 1, 64)
        assert need > 2 * 100000 * 2 * 64 * 4 and lib.a2v_linear_attention_workspace(0, 0, 0, 64, 2000, 16, 16, 64) == 0
        assert lib.a2v_linear_attention_bwd(0, p, p, p, p, p, p, p, st, p, None, None, None, None, 1, 100000, 2, 1, 64, 1.0, 0, p, need - 1, None) == -1
        assert lib.a2v_linear_attention_step(0, p, p, p, p, st, p, None, None, 4, 4, 2, 2, 64, 1.0, None) == -1
        assert lib.a2v_linear_attention_step(0, p, p, p, p, st, p, p, None, 3, 4, 2, 2, 64, 1.0, None) == -1
        assert lib.a2v_linear_attention_step(0, p, p, p, p, st, p, p, p, 1, 1 << 23, 2, 2, 64, 1.0, None) == -1
        assert lib.a2v_linear_attention_step(0, p + 4, p, p, p, st, p, p, p, 3, 4, 2, 2, 64, 1.0, None) == -1

        def rope(dtype=0, q=p, w=p, f=p, pos=p, ps=(C.c_longlong * 2)(4, 1), axes=3, sec=sec, HD=64, N=1):
            return lib.a2v_qk_norm_rope_fwd(dtype, q, p, p, p, st, w, p, f, pos, ps, axes, sec, 0, 1e-6, N, 4, 2, 2, HD, None)
        assert rope(dtype=2) == -2 and rope(q=None) == -1 and rope(q=p + 2) == -1 and rope(w=None) == -1 and rope(f=None) == -1 and rope(ps=None) == -1
        assert rope(axes=4) == -1 and rope(pos=None) == -1 and rope(sec=None) == -1 and rope(HD=32) == -1 and rope(sec=(C.c_int * 3)(16, 8, 7)) == -1 and rope(N=0) == 0
        assert lib.a2v_qk_norm_rope_bwd(0, p, p, p, p, p, p, st, p, p, p, p, p, None, None, 1, (C.c_int * 1)(32), 0, 1e-6, 1, 4, 2, 2, 64, None, 0, None) == -1


# ------------------------------------------------------------------------------------------------ norm + rotation on the GPU
@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from animal2vec_amd import ops as o
    return o


def rope_case(N, S, H, HK, HD, half, axes, dtype, first=0, seed=0):
    small = half // 4
    sections = (half - small * (axes - 1),) + (small,) * (axes - 1)
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(1, n)) for n in sections]).float()
    g = torch.Generator().manual_seed(seed + 9)
    pos = torch.randint(-50, 2000, (N, S, axes), generator=g, dtype=torch.int32)
    pos[..., 0] += first
    axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections))
    ang = (pos.double()[..., axis] * freq.double()).unsqueeze(2)
    qkv = rnd(N, S, H + 2 * HK, HD, seed=seed, dtype=dtype, scale=1.7)
    return sections, freq, pos, ang, qkv, 1 + 0.2 * rnd(HD, seed=seed + 1), 1 + 0.2 * rnd(HD, seed=seed + 2)


ROPE = [  # N, S, H, HK, HD, half, axes, interleaved, first
    (2, 37, 16, 16, 64, 32, 1, False, 0), (1, 1, 1, 1, 32, 16, 1, True, 7), (3, 129, 12, 4, 64, 16, 3, True, 0), (2, 50, 3, 1, 128, 64, 2, False, 17280000),
    (1, 700, 4, 2, 32, 8, 3, False, 2000000000), (5, 1, 8, 2, 128, 40, 3, True, -2000000000), (4, 141, 16, 16, 64, 24, 2, False, 0),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,S,H,HK,HD,half,axes,inter,first", ROPE)
def test_norm_rope_fwd_bwd(ops, N, S, H, HK, HD, half, axes, inter, first, dtype):
    import contextlib
    sections, freq, pos, ang, qkv, wq, wk = rope_case(N, S, H, HK, HD, half, axes, dtype, first)
    dqo, dko = rnd(N, S, H, HD, seed=5, dtype=dtype), rnd(N, S, HK, HD, seed=6, dtype=dtype)
    x = qkv.cuda()
    q, k = x[:, :, :H], x[:, :, H:H + HK]
    p = pos.cuda() if axes > 1 else pos[..., 0].contiguous().cuda()
    kw = dict(sections=sections, interleaved=inter, eps=1e-5)
    dwq, dwk = torch.full((HD,), 3.0).cuda(), torch.full((HD,), -2.0).cuda()
    with ops.half_library() if dtype == torch.float16 else contextlib.nullcontext():
        yq, yk = ops.qk_norm_rope_fwd(q, k, wq.cuda(), wk.cuda(), freq.cuda(), p, **kw)
        dq, dk = ops.qk_norm_rope_bwd(dqo.cuda(), dko.cuda(), q, k, wq.cuda(), wk.cuda(), freq.cuda(), p, dq_weight=dwq, dk_weight=dwk, **kw)
    assert torch.equal(x.cpu(), qkv)
    # an angle in 64 bits of a position below 2^31 is off by 2^31 2^-52: the sine's own error rules
    for got, gdx, gdw, xs, w, dy, base, name in ((yq, dq, dwq, qkv[:, :, :H], wq, dqo, 3.0, "q"), (yk, dk, dwk, qkv[:, :, H:H + HK], wk, dko, -2.0, "k")):
        xs, w, dy = xs.double(), w.double(), dy.double()
        a = torch.zeros_like(ang)
        one = lambda t: t.abs().amax(-1, keepdim=True).expand_as(t)       # noqa: E731  (a rotated pair mixes two channels)
        y = ref_norm_rope(xs, w, ang, inter, 1e-5)
        check(got, y, one(ref_norm_rope(xs.abs(), w.abs(), a, inter, 1e-5)), 2.0 ** -18, name)
        dx, dw = ref_norm_rope(xs, w, ang, inter, 1e-5, dy)
        r = (xs.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        # terms: r |g w| and r |x r| mean |g w x r| <= HD r max|g w| max|x r|
        gmax, xmax = dy.abs().amax(-1, keepdim=True) * 1.42 * w.abs().max(), (xs * r).abs().amax(-1, keepdim=True)
        check(gdx, dx, (r * gmax * (1 + xmax * xmax)).expand_as(dx), 2.0 ** -18, "d" + name)
        terms = (1.42 * dy.abs().amax(-1, keepdim=True) * (xs * r).abs()).sum((0, 1, 2))
        check(gdw, base + dw.sum((0, 1, 2)), base * base + terms, 2.0 ** -18, "dw" + name)


@gpu
def test_norm_rope_default_positions_in_place_and_slots(ops):
    """pos None counts rows; in place on a packed projection leaves v alone; gradients written into a packed gradient's slots, also onto
    the incoming ones; the same call twice gives the same bits"""
    N, S, H, HD = 2, 300, 4, 64
    qkv = rnd(N, S, 3, H, HD, seed=1, dtype=torch.bfloat16).cuda()
    wq, wk, f = 1 + 0.1 * rnd(HD, seed=2).cuda(), 1 + 0.1 * rnd(HD, seed=3).cuda(), ops.rope_inv_freq((HD // 2,))
    q, k, v = qkv.unbind(2)
    pos = torch.arange(S, dtype=torch.int32, device="cuda").expand(N, S)
    a = ops.qk_norm_rope_fwd(q, k, wq, wk, f)
    b = ops.qk_norm_rope_fwd(q, k, wq, wk, f, pos)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    work = qkv.clone()
    ops.qk_norm_rope_fwd(work[:, :, 0], work[:, :, 1], wq, wk, f, q_out=work[:, :, 0], k_out=work[:, :, 1])
    assert torch.equal(work[:, :, 0], a[0]) and torch.equal(work[:, :, 1], a[1]) and torch.equal(work[:, :, 2], v)
    dy = rnd(N, S, 3, H, HD, seed=4, dtype=torch.bfloat16).cuda()
    g = [torch.zeros(HD, device="cuda") for _ in range(4)]
    dq, dk = ops.qk_norm_rope_bwd(dy[:, :, 0], dy[:, :, 1], q, k, wq, wk, f, dq_weight=g[0], dk_weight=g[1])
    packed = dy.clone()
    ops.qk_norm_rope_bwd(packed[:, :, 0], packed[:, :, 1], q, k, wq, wk, f, dq_weight=g[2], dk_weight=g[3], dq=packed[:, :, 0], dk=packed[:, :, 1])
    assert torch.equal(packed[:, :, 0], dq) and torch.equal(packed[:, :, 1], dk) and torch.equal(packed[:, :, 2], dy[:, :, 2])
    assert torch.equal(g[0], g[2]) and torch.equal(g[1], g[3])
    e = ops.qk_norm_rope_fwd(q[:, :0], k[:, :0], wq, wk, f)
    assert e[0].shape == (N, 0, H, HD)


@gpu
def test_norm_rope_gradient_against_differences(ops):
    """fp32: (f(x + h d) - f(x - h d)) / 2h of the kernel's own forward against the kernel's gradient.  f is a sum of 480 products of
    size 1; with h = 2^-7 the cubic term is h^2 / 6 |f'''| ~ 1e-5 |f| and rounding 480 2^-24 / h ~ 4e-3 absolute worst, sqrt of that typical"""
    N, S, H, HD = 1, 5, 3, 32
    x, dy = rnd(N, S, 2 * H, HD, seed=1).cuda(), rnd(N, S, 2 * H, HD, seed=2).cuda()
    w, f = 1 + 0.1 * rnd(HD, seed=3).cuda(), ops.rope_inv_freq((HD // 2,))
    d, dw = rnd(N, S, 2 * H, HD, seed=4).cuda(), rnd(HD, seed=5).cuda()
    run = lambda x, w: sum((y.double() * g.double()).sum() for y, g in zip(ops.qk_norm_rope_fwd(x[:, :, :H], x[:, :, H:], w, w, f), (dy[:, :, :H], dy[:, :, H:])))   # noqa: E731
    gw = torch.zeros(2, HD, device="cuda")
    dq, dk = ops.qk_norm_rope_bwd(dy[:, :, :H], dy[:, :, H:], x[:, :, :H], x[:, :, H:], w, w, f, dq_weight=gw[0], dk_weight=gw[1])
    h = 2.0 ** -7
    num = (run(x + h * d, w) - run(x - h * d, w)) / (2 * h)
    ana = (torch.cat([dq, dk], 2).double() * d.double()).sum()
    assert abs(float(num - ana)) < 4e-3 + 1e-3 * abs(float(ana))
    num = (run(x, w + h * dw) - run(x, w - h * dw)) / (2 * h)
    ana = ((gw[0] + gw[1]).double() * dw.double()).sum()
    assert abs(float(num - ana)) < 4e-3 + 1e-3 * abs(float(ana))


# ------------------------------------------------------------------------------------------------ linear attention on the GPU
def lin_case(B, S, H, HK, HD, dtype, seed=0, state=True):
    q, k, v, do = (rnd(B, S, h, HD, seed=seed + i, dtype=dtype) for i, h in enumerate((H, HK, HK, H)))
    st, ds = (rnd(B, H, HD, HD, seed=seed + 7, scale=2.0), rnd(B, H, HD, HD, seed=seed + 8)) if state else (None, None)
    return q, k, v, do, st, ds


def lin_check(got, seqs, slopes, scale, dtype, H, HK, HD):
    """got: out, last, dq, dk, dv, first, each a list with one entry per sequence; seqs: (q, k, v, do, st, ds) of each"""
    for b, t in enumerate(seqs):
        t = [x.double() if x is not None else None for x in t]
        q, k, v, do, st, ds = t
        mag = [x.abs() if x is not None else None for x in t]
        want = ref_linear(q, k, v, slopes, scale, st, do, ds)
        size = ref_linear(mag[0], mag[1], mag[2], slopes, abs(scale), mag[4], mag[3], mag[5])
        c = c_of(dtype, q.shape[0], HD)
        for i, name in enumerate(("out", "last", "dq", "dk", "dv", "first")):
            if got[i] is not None:
                # states are results of the same sums (and never rounded below fp32)
                check(got[i][b], want[i], size[i], c, f"{name} of sequence {b} ({q.shape[0]} rows)")


LIN = [  # B, S, H, HK, HD
    (1, 1, 1, 1, 64), (2, 2, 2, 1, 32), (1, 31, 3, 3, 64), (2, 32, 2, 2, 128), (1, 33, 4, 1, 64), (3, 63, 2, 2, 64), (1, 64, 2, 1, 128), (2, 65, 2, 2, 64),
    (1, 127, 6, 2, 32), (2, 140, 4, 4, 64), (1, 200, 2, 2, 128), (1, 257, 3, 1, 64),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,HK,HD", LIN)
def test_linear_attention_fwd_bwd(ops, B, S, H, HK, HD, dtype):
    q, k, v, do, st, ds = lin_case(B, S, H, HK, HD, dtype)
    slopes, scale = alibi(H), HD ** -0.5
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    out, last = ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), state=d[4], want_state=True)
    dq, dk, dv, first = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5])
    assert torch.equal(d[4].cpu(), st)
    lin_check((out, last, dq, dk, dv, first), [(q[b], k[b], v[b], do[b], st[b], ds[b]) for b in range(B)], slopes, scale, dtype, H, HK, HD)
    # without states, another scale
    out, last = ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), scale=-0.7)
    assert last is None
    dq, dk, dv, first = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], scale=-0.7)
    assert first is None
    lin_check((out, None, dq, dk, dv, None), [(q[b], k[b], v[b], do[b], None, None) for b in range(B)], slopes, -0.7, dtype, H, HK, HD)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,HK,HD", [(1, 1500, 2, 1, 32), (2, 1025, 2, 2, 64), (1, 1100, 1, 1, 128)])
def test_linear_attention_split_over_the_axis(ops, B, S, H, HK, HD, dtype):
    """few heads, a long axis: segments (here of 4 HD rows) that start from the scanned states; slow decays so that they matter"""
    assert ops._L().a2v_linear_attention_workspace(ops.dt(torch.empty(0, dtype=dtype)), 0, 0, B, S, H, HK, HD) > 0
    q, k, v, do, st, ds = lin_case(B, S, H, HK, HD, dtype, seed=3)
    slopes, scale = torch.tensor([0.001, 0.02])[:H], HD ** -0.5
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    out, last = ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), state=d[4], want_state=True)
    got = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5])
    lin_check((out, last, *got), [(q[b], k[b], v[b], do[b], st[b], ds[b]) for b in range(B)], slopes, scale, dtype, H, HK, HD)
    again = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize("B,S,H,HD", [(64, 70, 16, 64), (34, 65, 32, 64), (64, 33, 16, 32), (256, 1, 4, 32)])
def test_neighbouring_heads_in_one_workgroup(ops, B, S, H, HD):
    """enough (sequence, head) pairs to give a workgroup two or four heads: the bits of the sequences one by one, and right ones"""
    q, k, v, do, st, ds = lin_case(B, S, H, H, HD, torch.bfloat16, seed=5)
    sl, scale = alibi(H), HD ** -0.5
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    got = (*ops.linear_attention_fwd(d[0], d[1], d[2], sl.cuda(), state=d[4], want_state=True),
           *ops.linear_attention_bwd(d[0], d[1], d[2], sl.cuda(), d[3], state=d[4], d_state=d[5]))
    for b in range(B):
        one = [t[b:b + 1] for t in d]
        want = (*ops.linear_attention_fwd(one[0], one[1], one[2], sl.cuda(), state=one[4].contiguous(), want_state=True),
                *ops.linear_attention_bwd(one[0], one[1], one[2], sl.cuda(), one[3], state=one[4].contiguous(), d_state=one[5].contiguous()))
        for x, y in zip(got, want):
            assert torch.equal(x[b], y[0])
    lin_check([t[:2] for t in got], [(q[b], k[b], v[b], do[b], st[b], ds[b]) for b in range(2)], sl, scale, torch.bfloat16, H, H, HD)


@gpu
@pytest.mark.parametrize("H,HD,far", [(32, 64, False), (32, 32, False), (2, 64, True)])
def test_neighbouring_heads_of_a_long_recording(ops, H, HD, far):
    """the same of a split axis, with rows outside the sequence, from a packed projection; heads too far apart for it take the other kernel"""
    S, lead, tail = (524320, 0, 0) if far else (40000, 40, 1000)
    cu = torch.tensor([lead, S - tail], dtype=torch.int32, device="cuda")
    sl = (alibi(H) + 0.5).cuda()
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(1, 3, H, S, HD, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = x.transpose(2, 3).unbind(1)
    if not far:
        q, k, v = x.permute(0, 3, 1, 2, 4).contiguous().unbind(2)
    out, last = ops.linear_attention_fwd(q, k, v, sl, cu_seqlens=cu, want_state=True)
    n = [t[0, S - tail - 300:S - tail].double().cpu() for t in (q, k, v)]     # e^(-0.5 * 200): what lies further back is below every rounding
    want = ref_linear(*n, sl.cpu(), HD ** -0.5)
    size = ref_linear(*(t.abs() for t in n), sl.cpu(), HD ** -0.5)
    check(out[0, S - tail - 100:S - tail], want[0][-100:], size[0][-100:] + 1.0, 2.0 ** -14, "last rows")
    check(last[0], want[1], size[1], c_of(torch.float32, 300, HD), "state")
    assert not out[0, :lead].any() and not out[0, S - tail:].any()
    dense, _ = ops.linear_attention_fwd(*(t[:, lead:S - tail].contiguous() for t in (q, k, v)), sl)
    n = [t[0, lead:lead + 200].double().cpu() for t in (q, k, v)]
    want = ref_linear(*n, sl.cpu(), HD ** -0.5)
    size = ref_linear(*(t.abs() for t in n), sl.cpu(), HD ** -0.5)
    for t in (out[0, lead:lead + 200], dense[0, :200]):
        check(t, want[0], size[0], 2.0 ** -14, "first rows")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,lead,tail,H,HK,HD", [((5, 0, 64, 1, 130, 0), 3, 9, 4, 2, 64), ((0,), 0, 4, 2, 2, 32), ((700, 3, 0, 1200, 256), 17, 300, 2, 1, 32), ((40, 90), 0, 0, 2, 2, 128)])
def test_linear_attention_packed(ops, lens, lead, tail, H, HK, HD, dtype):
    """sequences of any length side by side, empty ones handing their state on; NaN in the rows outside of them"""
    T, B = lead + sum(lens) + tail, len(lens)
    q, k, v, do, _, _ = lin_case(1, T, H, HK, HD, dtype, seed=11, state=False)
    st, ds = rnd(B, H, HD, HD, seed=21, scale=2.0), rnd(B, H, HD, HD, seed=22)
    cu = torch.tensor([lead] + list(lens)).cumsum(0).to(torch.int32)
    a, e = int(cu[0]), int(cu[-1])
    for t in (q, k, v, do):
        t[:, :a] = float("nan")
        t[:, e:] = float("inf")
    slopes, scale = alibi(H, 0.003), HD ** -0.5
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    out, last = ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), state=d[4], want_state=True, cu_seqlens=cu.cuda())
    dq, dk, dv, first = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5], cu_seqlens=cu.cuda())
    cut = lambda t: [t[0, cu[b]:cu[b + 1]] for b in range(B)]     # noqa: E731
    lin_check((cut(out), last, cut(dq), cut(dk), cut(dv), first), [(cut(q)[b], cut(k)[b], cut(v)[b], cut(do)[b], st[b], ds[b]) for b in range(B)],
              slopes, scale, dtype, H, HK, HD)
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.equal(last[b].cpu(), st[b]) and torch.equal(first[b].cpu(), ds[b])
    for t in (out, dq, dk, dv):
        assert not t[:, :a].any() and not t[:, e:].any()
    # the caller's own results: rows outside are left as they were
    mine = [torch.full_like(t, 7.0) for t in (out, dq, dk, dv)]
    ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), state=d[4], cu_seqlens=cu.cuda(), out=mine[0])
    ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5], cu_seqlens=cu.cuda(), dq=mine[1], dk=mine[2], dv=mine[3])
    for t, m in zip((out, dq, dk, dv), mine):
        assert torch.equal(t[:, a:e], m[:, a:e]) and bool((m[:, :a] == 7).all()) and bool((m[:, e:] == 7).all())


@gpu
def test_linear_attention_wrong_offsets_stay_inside(ops):
    """descending and out-of-range offsets are clamped: whatever comes out, nothing outside the tensors is touched and later calls work"""
    T, H, HD = 300, 2, 64
    guard = torch.full((3 * T, H, HD), 5.0, device="cuda", dtype=torch.bfloat16)
    q, k, v, _, _, _ = (t.cuda() if t is not None else None for t in lin_case(1, T, H, H, HD, torch.bfloat16, state=False))
    for cu in ([0, 200, 100, 300], [-50, 20, 4000], [2 ** 31 - 1, 0], [300, 300]):
        ops.linear_attention_fwd(q, k, v, alibi(H).cuda(), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), out=guard[T:2 * T].unsqueeze(0), want_state=True)
        torch.cuda.synchronize()
        assert bool((guard[:T] == 5).all()) and bool((guard[2 * T:] == 5).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_attention_extreme_decays(ops, dtype):
    """no decay, complete forgetting (infinity: out = scale (q.k) v), and decays that underflow within a chunk"""
    B, S, H, HD = 1, 150, 4, 64
    q, k, v, do, st, ds = lin_case(B, S, H, H, HD, dtype, seed=31)
    slopes = torch.tensor([0.0, float("inf"), 50.0, 1e-6])
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    out, last = ops.linear_attention_fwd(d[0], d[1], d[2], slopes.cuda(), state=d[4], want_state=True)
    got = ops.linear_attention_bwd(d[0], d[1], d[2], slopes.cuda(), d[3], state=d[4], d_state=d[5])
    lin_check((out, last, *got), [(q[0], k[0], v[0], do[0], st[0], ds[0])], slopes, HD ** -0.5, dtype, H, H, HD)
    o, s = ops.linear_attention_fwd(d[0][:, :0], d[1][:, :0], d[2][:, :0], slopes.cuda(), state=d[4], want_state=True)
    assert o.shape == (B, 0, H, HD) and torch.equal(s.cpu(), st)


@gpu
def test_linear_attention_non_finite_rows_do_not_reach_the_past(ops):
    """a NaN key or an infinite value leaves the rows of earlier blocks (64 rows) and other sequences as they were"""
    S, H, HD = 200, 2, 64
    q, k, v, _, _, _ = (t.cuda() if t is not None else None for t in lin_case(2, S, H, H, HD, torch.bfloat16, state=False))
    ref, _ = ops.linear_attention_fwd(q, k, v, alibi(H).cuda())
    k2, v2 = k.clone(), v.clone()
    k2[0, 140, 1, 3] = float("nan")
    v2[0, 150, 1, 9] = float("inf")
    out, _ = ops.linear_attention_fwd(q, k2, v2, alibi(H).cuda())
    assert torch.equal(out[0, :128], ref[0, :128]) and torch.equal(out[1], ref[1]) and torch.equal(out[0, :, 0], ref[0, :, 0])
    assert bool(torch.isnan(out[0, 140:, 1]).any())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,H,HK,HD,pool", [(1, 1, 1, 64, 0), (5, 4, 2, 32, 0), (7, 3, 3, 128, 11), (300, 2, 1, 64, 301)])
def test_linear_attention_step(ops, N, H, HK, HD, pool, dtype):
    qkv = rnd(N, H + 2 * HK, HD, seed=1, dtype=dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    P = pool or N + 2
    state = rnd(P, H, HD, HD, seed=2)
    slots = torch.randperm(P, generator=torch.Generator().manual_seed(3))[:N].to(torch.int32) if pool else None
    sd, x = state.cuda(), qkv.cuda()
    with ops.half_library() if dtype == torch.float16 else contextlib.nullcontext():
        out = ops.linear_attention_step(x[:, :H], x[:, H:H + HK], x[:, H + HK:], alibi(H).cuda(), sd, slots=slots.cuda() if pool else None, scale=0.9)
    for n in range(min(N, 40)):
        s = int(slots[n]) if pool else n
        want = ref_linear(q[n:n + 1].double(), k[n:n + 1].double(), v[n:n + 1].double(), alibi(H), 0.9, state[s].double())
        size = ref_linear(q[n:n + 1].double().abs(), k[n:n + 1].double().abs(), v[n:n + 1].double().abs(), alibi(H), 0.9, state[s].double().abs())
        check(out[n:n + 1], want[0], size[0], (HD + 16) * 2.0 ** -24, f"row {n}")
        check(sd[s], want[1], size[1], 4 * 2.0 ** -24, f"state of row {n}")
    touched = set(int(s) for s in slots) if pool else set(range(N))
    for s in set(range(P)) - touched:
        assert torch.equal(sd[s].cpu(), state[s])


@gpu
def test_linear_attention_step_repeated_and_missing_slots(ops):
    """rows of one slot are successive tokens in row order; a slot outside the pool gives zeros and touches nothing"""
    N, H, HK, HD, P = 9, 4, 2, 64, 4
    q, k, v = rnd(N, H, HD, seed=1).cuda(), rnd(N, HK, HD, seed=2).cuda(), rnd(N, HK, HD, seed=3).cuda()
    slots = [2, -1, 0, 2, 7, 2, 0, 1, 2]
    state = rnd(P, H, HD, HD, seed=4).cuda()
    a, b = state.clone(), state.clone()
    out = ops.linear_attention_step(q, k, v, alibi(H).cuda(), a, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    for n, s in enumerate(slots):
        if 0 <= s < P:
            o = ops.linear_attention_step(q[n:n + 1], k[n:n + 1], v[n:n + 1], alibi(H).cuda(), b[s:s + 1])
            assert torch.equal(o[0], out[n]), n
        else:
            assert not out[n].any()
    assert torch.equal(a, b) and torch.equal(a[3], state[3])
    assert ops.linear_attention_step(q[:0], k[:0], v[:0], alibi(H).cuda(), a).shape == (0, H, HD)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_single_tokens_is_the_whole(ops, dtype):
    """a run as it is used: packed projection -> norm + rotation in place -> chunked prompt -> single tokens, against the recurrence over
    everything; the rotated q and k are compared first and then taken as they are"""
    N, S, tail, H, HD = 2, 210, 6, 4, 64
    qkv = rnd(N, S + tail, 3, H, HD, seed=1, dtype=dtype).cuda()
    wq, wk, f = 1 + 0.1 * rnd(HD, seed=2).cuda(), 1 + 0.1 * rnd(HD, seed=3).cuda(), ops.rope_inv_freq((16, 8, 8))
    pos = torch.randint(0, 3000, (N, S + tail, 3), generator=torch.Generator().manual_seed(4), dtype=torch.int32).cuda()
    slopes = alibi(H).cuda()
    kw = dict(sections=(16, 8, 8))
    whole = ops.qk_norm_rope_fwd(qkv[:, :, 0], qkv[:, :, 1], wq, wk, f, pos, **kw)
    work = qkv.clone()
    q, k, v = work.unbind(2)
    ops.qk_norm_rope_fwd(q[:, :S], k[:, :S], wq, wk, f, pos[:, :S], q_out=q[:, :S], k_out=k[:, :S], **kw)
    out, state = ops.linear_attention_fwd(q[:, :S], k[:, :S], v[:, :S], slopes, want_state=True)
    outs = [out]
    for t in range(S, S + tail):
        ops.qk_norm_rope_fwd(q[:, t:t + 1], k[:, t:t + 1], wq, wk, f, pos[:, t:t + 1], q_out=q[:, t:t + 1], k_out=k[:, t:t + 1], **kw)
        outs.append(ops.linear_attention_step(q[:, t], k[:, t], v[:, t], slopes, state).unsqueeze(1))
    assert torch.equal(q, whole[0]) and torch.equal(k, whole[1])
    out = torch.cat(outs, 1)
    qc, kc, vc = (t.double().cpu() for t in (q, k, v))
    for n in range(N):
        want = ref_linear(qc[n], kc[n], vc[n], alibi(H), HD ** -0.5)
        size = ref_linear(qc[n].abs(), kc[n].abs(), vc[n].abs(), alibi(H), HD ** -0.5)
        check(out[n], want[0], size[0], c_of(dtype, S + tail, HD), f"out {n}")
        check(state[n], want[1], size[1], c_of(dtype, S + tail, HD), f"state {n}")


@gpu
def test_linear_attention_gradient_against_differences(ops):
    """fp32: central differences of the kernel's own forward are exact for a function linear in q, in v and in the state (and bilinear
    along all of them at once up to h^2): rounding 2^-24 A / h with A ~ 40 x 96 terms of size 1 and h = 2^-5 stays below 2e-2 absolute"""
    B, S, H, HD = 1, 40, 3, 32
    q, k, v, do, st, ds = (t.cuda() for t in lin_case(B, S, H, H, HD, torch.float32, seed=5))
    slopes = alibi(H).cuda()

    def f(q, k, v, st):
        o, s = ops.linear_attention_fwd(q, k, v, slopes, state=st, want_state=True)
        return (o.double() * do.double()).sum() + (s.double() * ds.double()).sum()
    grads = ops.linear_attention_bwd(q, k, v, slopes, do, state=st, d_state=ds)
    args, h = [q, k, v, st], 2.0 ** -5
    for i, g in enumerate(grads):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(50 + i)).cuda()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        num, ana = (f(*up) - f(*down)) / (2 * h), (g.double() * d.double()).sum()
        assert abs(float(num - ana)) < 2e-2 + 1e-4 * abs(float(ana)), (i, float(num), float(ana))


@gpu
def test_strided_operands_and_packed_gradients(ops):
    """views of a packed projection in, slots of a packed gradient out, k and v broadcast over the batch (stride 0): the same bits as
    contiguous operands"""
    N, S, H, HD = 3, 100, 4, 64
    qkv, do = rnd(N, S, 3, H, HD, seed=1, dtype=torch.bfloat16).cuda(), rnd(N, S, H, HD, seed=2, dtype=torch.bfloat16).cuda()
    q, k, v = qkv.unbind(2)
    sl = alibi(H).cuda()
    a = ops.linear_attention_fwd(q, k, v, sl)[0]
    b = ops.linear_attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), sl)[0]
    assert torch.equal(a, b)
    g = torch.full_like(qkv, 9.0)
    ops.linear_attention_bwd(q, k, v, sl, do, dq=g[:, :, 0], dk=g[:, :, 1], dv=g[:, :, 2])
    w = ops.linear_attention_bwd(q.contiguous(), k.contiguous(), v.contiguous(), sl, do)
    assert all(torch.equal(g[:, :, i], w[i]) for i in range(3))
    ke, ve = k[:1].expand(N, S, H, HD), v[:1].expand(N, S, H, HD)
    assert torch.equal(ops.linear_attention_fwd(q, ke, ve, sl)[0], ops.linear_attention_fwd(q, ke.contiguous(), ve.contiguous(), sl)[0])
    e, c = ops.linear_attention_bwd(q, ke, ve, sl, do), ops.linear_attention_bwd(q, ke.contiguous(), ve.contiguous(), sl, do)
    assert all(torch.equal(x, y) for x, y in zip(e[:3], c[:3]))
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)          # (N, H, S, HD) in memory
    assert torch.equal(ops.linear_attention_fwd(heads_first, k, v, sl)[0], a)


@gpu
def test_streams_and_captured_graphs(ops):
    """forward, backward and step captured in two graphs of their own and replayed with eager calls in between: every replay equals the
    eager result (workspaces come from the graph's pool, nothing is shared); a call on a side stream runs there"""
    S, H, HD = 1500, 2, 32
    dev = [t.cuda() for t in lin_case(1, S, H, H, HD, torch.bfloat16, seed=2)]
    q, k, v, do, st, ds = dev
    sl, f = alibi(H).cuda(), ops.rope_inv_freq((HD // 2,))
    w = torch.ones(HD, device="cuda")
    gw = torch.zeros(2, HD, device="cuda")

    def once(pool):
        yq, yk = ops.qk_norm_rope_fwd(q, k, w, w, f)
        out, last = ops.linear_attention_fwd(yq, yk, v, sl, state=st, want_state=True)
        dq, dk, dv, first = ops.linear_attention_bwd(yq, yk, v, sl, do, state=st, d_state=ds)
        dq, dk = ops.qk_norm_rope_bwd(dq, dk, q, k, w, w, f, dq_weight=gw[0], dk_weight=gw[1])
        o1 = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], sl, pool)
        return out, last, dq, dk, dv, first, o1
    pools = [st.clone() for _ in range(3)]
    want = [t.clone() for t in once(pools[0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once(pools[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for i in range(2):
        pool = st.clone()
        with torch.cuda.stream(side):
            once(pool)
        side.synchronize()
        pool.copy_(st)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = once(pool)
        graphs.append((g, res, pool))
    for rep in range(3):
        for g, res, pool in graphs:
            for t in res:
                t.zero_()
            pool.copy_(st)
            g.replay()
            eager = once(pools[2].copy_(st))
            torch.cuda.synchronize()
            for a, b, c in zip(want, res, eager):
                assert torch.equal(a, b) and torch.equal(a, c)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_replays_follow_the_offsets_on_the_device(ops, dtype):
    """a captured packed forward and backward of shared heads, replayed with other inputs and other sequences in the same buffers: each
    replay equals an eager call, rows outside every sequence are zeros again"""
    T, H, HK, HD = 1300, 4, 2, 64
    lay = [(0, 700, 700, 1300), (40, 41, 900, 1200), (0, 0, 1300, 1300), (1299, 1299, 1299, 1299)]
    q, k, v, do = (rnd(1, T, h, HD, seed=i, dtype=dtype).cuda() for i, h in enumerate((H, HK, HK, H)))
    cu, sl = torch.tensor(lay[0], dtype=torch.int32, device="cuda"), alibi(H, 0.01).cuda()
    st, ds = (rnd(3, H, HD, HD, seed=i).cuda() for i in (7, 8))

    def once():
        out, last = ops.linear_attention_fwd(q, k, v, sl, state=st, cu_seqlens=cu, want_state=True)
        return (out, last, *ops.linear_attention_bwd(q, k, v, sl, do, state=st, d_state=ds, cu_seqlens=cu))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = once()
    for i, c in enumerate(lay + lay[:1]):
        cu.copy_(torch.tensor(c, dtype=torch.int32))
        q.copy_(rnd(1, T, H, HD, seed=20 + i, dtype=dtype))
        for t in res:
            t.fill_(9.0)
        g.replay()
        want = once()
        torch.cuda.synchronize()
        for a, b in zip(res, want):
            assert torch.equal(a, b)
        for t in (res[0], res[2], res[3], res[4]):
            assert not t[0, :c[0]].any() and not t[0, c[-1]:].any()


@gpu
def test_calls_on_two_streams_and_from_two_threads(ops):
    """calls in flight at the same time have their own workspaces"""
    H, HD = 4, 64
    sl = alibi(H).cuda()
    sets = [[t.cuda() for t in lin_case(1, S, H, H, HD, torch.bfloat16, seed=S)] for S in (3000, 2500)]

    def call(x, n=1):
        for _ in range(n):
            r = ops.linear_attention_fwd(x[0], x[1], x[2], sl, state=x[4], want_state=True) + \
                ops.linear_attention_bwd(x[0], x[1], x[2], sl, x[3], state=x[4], d_state=x[5])
        return r
    want = [call(x) for x in sets]
    torch.cuda.synchronize()
    streams, got, errors = [torch.cuda.Stream() for _ in sets], [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(streams[i]):
                got[i] = call(sets[i], 20)
        except Exception as e:      # noqa: BLE001 (shown below)
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
@pytest.mark.parametrize("N,H,HD", [(64, 16, 64), (2, 16, 64), (3, 2, 128)])
def test_rows_far_apart(ops, N, H, HD):
    """rows 60 MiB apart: offsets inside a chunk pass 31 bits; results in such rows as well, and the bytes between them left alone"""
    S, row = 33, 30 << 20
    base = torch.zeros((S - 1) * row + 4 * N * H * HD, dtype=torch.bfloat16, device="cuda")
    view = lambda i: base.as_strided((N, S, H, HD), (4 * H * HD, row, HD, 1), i * H * HD)          # noqa: E731
    q, k, v, out = (view(i) for i in range(4))
    g = torch.Generator("cuda").manual_seed(1)
    for t in (q, k, v):
        t.copy_(torch.randn(N, S, H, HD, generator=g, device="cuda"))
    sl = alibi(H).cuda()
    want, _ = ops.linear_attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), sl)
    kept = [t.clone() for t in (q, k, v)]
    ops.linear_attention_fwd(q, k, v, sl, out=out)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(kept, (q, k, v)))
    assert not base[4 * N * H * HD:row].any()
    do = rnd(N, S, H, HD, seed=4, dtype=torch.bfloat16).cuda()
    grads = ops.linear_attention_bwd(*(t.contiguous() for t in (q, k, v)), sl, do)
    for a, b in zip(grads[:3], ops.linear_attention_bwd(q, k, v, sl, do)):
        assert torch.equal(a, b)


@gpu
def test_long_offsets_pass_32_bits(ops):
    """a packed buffer of more than 2^31 elements: the last rows are as right as the first ones (addresses are formed in 64 bits)"""
    H, HD, W = 2, 64, 60 * 64
    S = 560032                                                   # S * W = 2.15e9 elements
    base = torch.empty(S, W, dtype=torch.bfloat16, device="cuda")
    view = base.view(1, S, 60, HD)
    assert base.numel() > 2 ** 31
    q, k, v = view[:, :, 0:H], view[:, :, 20:20 + H], view[:, :, 58:58 + H]
    for i, t in enumerate((q, k, v)):
        t.copy_(torch.randn(1, S, H, HD, generator=torch.Generator("cuda").manual_seed(i), device="cuda").to(torch.bfloat16))
    sl = torch.tensor([0.5, 1.0], device="cuda")
    out, _ = ops.linear_attention_fwd(q, k, v, sl)
    tail = 300                                                   # e^(-0.5 * 200): what lies further back is below every rounding
    n = [t[0, -tail:].double().cpu() for t in (q, k, v)]
    want = ref_linear(*n, sl.cpu(), HD ** -0.5)
    size = ref_linear(*(t.abs() for t in n), sl.cpu(), HD ** -0.5)
    check(out[0, -100:], want[0][-100:], size[0][-100:] + 1.0, 2.0 ** -14, "last rows")
    ref = ops.qk_norm_rope_fwd(q[:, -5:].contiguous(), k[:, -5:].contiguous(), torch.ones(HD, device="cuda"), torch.ones(HD, device="cuda"), ops.rope_inv_freq((32,)),
                               torch.arange(S - 5, S, dtype=torch.int32, device="cuda").view(1, 5))
    got = ops.qk_norm_rope_fwd(q, k, torch.ones(HD, device="cuda"), torch.ones(HD, device="cuda"), ops.rope_inv_freq((32,)))
    assert torch.equal(got[0][:, -5:], ref[0]) and torch.equal(got[1][:, -5:], ref[1])
