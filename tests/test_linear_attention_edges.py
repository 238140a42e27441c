"""Linear attention where it can go wrong and random inputs do not show it: the bits of what is kept between the products, and what the
tests beside these (test_linear_attention.py, whose references and bounds are used here) leave out."""
import pytest
import torch

from test_linear_attention import U, alibi, c_of, check, lin_case, ref_linear, rnd

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from animal2vec_amd import ops as o
    return o


# ------------------------------------------------------------------------------------------------ bits
# Two terms of size A that are equal up to 2^-12 are subtracted: the result's own rounding, u 2^-12 A = 2^-20 A in bf16, is below what a
# term loses if it is kept in 16 bits (up to 2^-16 A), and above what is lost in 32 (c A, c counted at each test).
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_keep_32_bits(ops, dtype):
    """v is 1 and -1 in two rows whose scores are equal up to 2^-12.  A score: HD products added in 32 bits, its weight and scale 8 more
    roundings: c = (HD + 8) 2^-24"""
    B, H, HD = 64, 4, 32
    q, k = rnd(B, 2, H, HD, seed=1, dtype=dtype), rnd(B, 2, H, HD, seed=2, dtype=dtype).abs()
    q = q.abs() + torch.tensor(0.5, dtype=dtype)
    k[:, 1] = k[:, 0]
    k[:, 0, :, 0], k[:, 1, :, 0] = 2.0 ** -8, 0.0            # q_0 2^-8 of about 20
    v = torch.zeros(B, 2, H, HD, dtype=dtype)
    v[:, 0], v[:, 1] = 1.0, -1.0
    sl = torch.zeros(H)
    out, _ = ops.linear_attention_fwd(q.cuda(), k.cuda(), v.cuda(), sl.cuda())
    for b in range(B):
        want = ref_linear(q[b].double(), k[b].double(), v[b].double(), sl, HD ** -0.5)[0]
        size = ref_linear(q[b].double(), k[b].double(), v[b].double().abs(), sl, HD ** -0.5)[0]
        assert float((want[1].abs() / size[1]).max()) < 2.0 ** -10
        check(out[b], want, size, (HD + 8) * 2.0 ** -24, f"sequence {b}")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,HD,B", [(4, 32, 8), (2, 64, 8), (2, 128, 8), (16, 64, 64)])
def test_the_state_that_rows_read_keeps_32_bits(ops, dtype, H, HD, B):
    """a row with q = (1, -1, 0 ...) and no key reads the difference of two rows of the state.  Decay, scale and sum of two terms: 8
    roundings.  Forward (out) and backward (dv and dk of a row with nothing of its own read D)"""
    st = rnd(B, H, HD, HD, seed=1, scale=2.0)
    st[:, :, 1] = st[:, :, 0] * (1 + 2.0 ** -12)
    q = torch.zeros(B, 1, H, HD, dtype=dtype)
    q[..., 0], q[..., 1] = 1.0, -1.0
    z, sl = torch.zeros_like(q), alibi(H)
    out, last = ops.linear_attention_fwd(q.cuda(), z.cuda(), z.cuda(), sl.cuda(), state=st.cuda(), want_state=True)
    dq, dk, dv, first = ops.linear_attention_bwd(z.cuda(), q.cuda(), z.cuda(), sl.cuda(), z.cuda(), d_state=st.cuda(), state=st.cuda())
    _, dk2, _, _ = ops.linear_attention_bwd(z.cuda(), z.cuda(), q.cuda(), sl.cuda(), z.cuda(), d_state=st.transpose(2, 3).contiguous().cuda())
    lam = torch.exp(-sl.double())[:, None]
    want = (st[:, :, 0].double() - st[:, :, 1].double()).unsqueeze(1)
    size = (st[:, :, 0].double().abs() + st[:, :, 1].double().abs()).unsqueeze(1)
    c = 8 * 2.0 ** -24
    check(out, lam * want * HD ** -0.5, lam * size * HD ** -0.5, c, "out")
    check(dv, want, size, c, "dv")
    check(dk2, want, size, c, "dk")
    assert not dq.any()
    check(last, st.double() * lam.unsqueeze(-1), st.double().abs() * lam.unsqueeze(-1), c, "last")
    check(first, st.double() * lam.unsqueeze(-1), st.double().abs() * lam.unsqueeze(-1), c, "first")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,HD,B", [(4, 32, 2), (2, 64, 2), (2, 128, 2), (16, 64, 64)])
def test_the_values_that_a_state_sums_keep_32_bits(ops, dtype, H, HD, B):
    """two rows whose keys are 1 and -1 and whose values are equal, a step of exp(-2^-12) apart, read a block later.  Two
    powers to an ulp (4 half steps), a product of powers and one with the value for each of two terms (4), the parts' products added (6), two
    more behind them: 16 roundings.  In the backward pass the same through dv and dk, without a gradient of the last state"""
    S, sl = 70, torch.full((H,), 2.0 ** -12)
    x = rnd(B, 1, H, HD, seed=1, dtype=dtype)
    one = torch.zeros(B, S, H, HD, dtype=dtype)
    e = lambda r, w: one.clone().index_fill_(1, torch.tensor(r), 1.0) * torch.tensor(w, dtype=dtype)       # noqa: E731
    unit = torch.zeros(HD, dtype=dtype)
    unit[3] = 1.0
    # forward: keys e_3, -e_3 at rows 4 and 5, q = e_3 at row 69
    k = (e([4], 1.0) - e([5], 1.0)) * unit
    q = e([69], 1.0) * unit
    v = (e([4], 1.0) + e([5], 1.0)) * x
    dev = lambda *t: [y.cuda() for y in t]                    # noqa: E731
    out, _ = ops.linear_attention_fwd(*dev(q, k, v, sl), scale=1.0)
    w = torch.exp(-(2.0 ** -12) * torch.tensor([65.0, 64.0], dtype=torch.float64))
    c = 16 * 2.0 ** -24
    check(out[:, 69:], x.double() * (w[0] - w[1]), x.double().abs() * w.sum(), c, "out")
    # backward: q e_3, -e_3 at rows 65 and 64 with gradients x; row 0 has k = e_3 (dv) or v = anything (dk)
    q2, do = (e([65], 1.0) - e([64], 1.0)) * unit, (e([64], 1.0) + e([65], 1.0)) * x
    _, _, dv, _ = ops.linear_attention_bwd(*dev(q2, e([0], 1.0) * unit, one, sl, do), scale=1.0)
    w = torch.exp(-(2.0 ** -12) * torch.tensor([65.0, 64.0], dtype=torch.float64))
    check(dv[:, :1], x.double() * (w[0] - w[1]), x.double().abs() * w.sum(), c, "dv")
    # dk_0 = sum_t w_t (v_0 . do_t) q_t: do e_3, -e_3 with q = x
    _, dk, _, _ = ops.linear_attention_bwd(*dev(do, one, e([0], 1.0) * unit, sl, q2), scale=1.0)
    check(dk[:, :1], x.double() * (w[0] - w[1]), x.double().abs() * w.sum(), c, "dk")


@gpu
@pytest.mark.parametrize("B,S,H,HK,HD", [(1, 33, 4, 2, 64), (2, 140, 4, 4, 64), (1, 257, 2, 1, 128), (1, 200, 4, 4, 32)])
def test_states_of_bf16_calls_are_fp32_results(ops, B, S, H, HK, HD):
    """the state and its gradient within the bound of fp32 calls"""
    q, k, v, do, st, ds = lin_case(B, S, H, HK, HD, torch.bfloat16, seed=41)
    sl = alibi(H)
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    _, last = ops.linear_attention_fwd(d[0], d[1], d[2], sl.cuda(), state=d[4], want_state=True)
    first = ops.linear_attention_bwd(d[0], d[1], d[2], sl.cuda(), d[3], state=d[4], d_state=d[5])[3]
    for b in range(B):
        t = [x[b].double() for x in (q, k, v)] + [sl, HD ** -0.5] + [x[b].double() for x in (st, do, ds)]
        want, size = ref_linear(*t), ref_linear(*(x.abs() if torch.is_tensor(x) and x is not sl else x for x in t))
        check(last[b], want[1], size[1], c_of(torch.float32, S, HD), "last")
        check(first[b], want[5], size[5], c_of(torch.float32, S, HD), "first")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,H,HK,HD", [(2300, 2, 1, 64), (4400, 1, 1, 128), (2300, 2, 2, 64)])
def test_backward_through_the_scan(ops, dtype, S, H, HK, HD):
    """more than 16 segments (of 2 HD rows): every segment starts from the scanned states, dk from the transposes of dv's"""
    q, k, v, do, st, ds = lin_case(1, S, H, HK, HD, dtype, seed=13)
    sl, scale = torch.tensor([0.001, 0.02])[:H], HD ** -0.5
    d = [t.cuda() for t in (q, k, v, do, st, ds)]
    got = (*ops.linear_attention_fwd(d[0], d[1], d[2], sl.cuda(), state=d[4], want_state=True),
           *ops.linear_attention_bwd(d[0], d[1], d[2], sl.cuda(), d[3], state=d[4], d_state=d[5]))
    t = [x[0].double() for x in (q, k, v)] + [sl, scale] + [x[0].double() for x in (st, do, ds)]
    want, size = ref_linear(*t), ref_linear(*(x.abs() if torch.is_tensor(x) and x is not sl else x for x in t))
    c = c_of(dtype, S, HD)
    for g, w, m, name in zip(got, want, size, ("out", "last", "dq", "dk", "dv", "first")):
        check(g[0], w, m, c, name)


# ------------------------------------------------------------------------------------------------ values that are not finite
# which elements of which result a value that is not finite reaches: (its own row and those behind or in front of it, or its own alone;
# its own channel or all)
REACH = {"q": dict(out=("own", "all"), dk=("front", "channel"), dv=("front", "all")),
         "k": dict(out=("behind", "all"), dq=("behind", "channel"), dv=("own", "all")),
         "v": dict(out=("behind", "channel"), dq=("behind", "all"), dk=("own", "all")),
         "d_out": dict(dq=("own", "all"), dk=("front", "all"), dv=("front", "channel"))}


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,HD,row", [(2, 75, 2, 32, 40), (2, 75, 2, 64, 74), (1, 70, 3, 128, 13), (1, 45, 2, 64, 44), (64, 70, 16, 64, 37), (64, 70, 32, 32, 33), (1, 700, 2, 64, 300),
                                          (1, 33, 2, 64, 0), (1, 1300, 1, 32, 1295)])
def test_values_that_are_not_finite_reach_what_the_formula_says(ops, B, S, H, HD, row, dtype):
    """one NaN or infinity in q, k, v or d_out: everything that it does not reach has the bits that it has beside a finite value, also in the
    same block of rows and beside copies of a last row; everything that it reaches is not finite"""
    q, k, v, do, _, _ = lin_case(B, S, H, H, HD, dtype, seed=51, state=False)
    dev = {n: t.cuda() for n, t in (("q", q), ("k", k), ("v", v), ("d_out", do))}
    sl, b, h, ch = (alibi(H) * 0.05).cuda(), B - 1, H - 1, HD - 3

    def run(d):
        o = ops.linear_attention_fwd(d["q"], d["k"], d["v"], sl, want_state=True)
        g = ops.linear_attention_bwd(d["q"], d["k"], d["v"], sl, d["d_out"])
        return dict(out=o[0], last=o[1], dq=g[0], dk=g[1], dv=g[2])
    clean = run(dev)
    for name, bad in (("q", "nan"), ("k", "inf"), ("v", "nan"), ("v", "inf"), ("v", "-inf"), ("k", "nan"), ("d_out", "-inf"), ("q", "inf"), ("d_out", "nan")):
        x = dev[name].clone()
        x[b, row, h, ch] = float(bad)
        got = run({**dev, name: x})
        for res in ("out", "dq", "dk", "dv"):
            hit = torch.zeros_like(clean[res], dtype=torch.bool)
            if res in REACH[name]:
                where, what = REACH[name][res]
                rows = slice(row, row + 1) if where == "own" else slice(row, None) if where == "behind" else slice(0, row + 1)
                hit[b, rows, h, ch if what == "channel" else slice(None)] = True
            assert torch.equal(got[res][~hit], clean[res][~hit]), (name, bad, res)
            assert not torch.isfinite(got[res][hit]).any(), (name, bad, res)
        hit = torch.zeros_like(clean["last"], dtype=torch.bool)
        if name == "k":
            hit[b, h, ch] = True
        if name == "v":
            hit[b, h, :, ch] = True
        assert torch.equal(got["last"][~hit], clean["last"][~hit]) and not torch.isfinite(got["last"][hit]).any(), (name, bad)


@gpu
def test_values_that_are_not_finite_in_packed_sequences(ops):
    """a NaN in the last row of a sequence, which the rows that its last block lacks are copies of, and in the first of the next one: the rows
    of the one in front and behind, and the other heads' share of a shared head's gradient, stay as they are"""
    T, H, HK, HD = 190, 4, 2, 64
    q, k, v, do = (rnd(1, T, h, HD, seed=i, dtype=torch.bfloat16).cuda() for i, h in enumerate((H, HK, HK, H)))
    cu, sl = torch.tensor([0, 45, 112, 190], dtype=torch.int32, device="cuda"), (alibi(H) * 0.1).cuda()
    out = ops.linear_attention_fwd(q, k, v, sl, cu_seqlens=cu)[0]
    grads = ops.linear_attention_bwd(q, k, v, sl, do, cu_seqlens=cu)[:3]
    x, d = v.clone(), do.clone()
    x[0, 111, 1, 7], x[0, 112, 0, 5] = float("inf"), float("nan")
    d[0, 44, 3, 9], d[0, 45, 0, 2] = float("nan"), float("inf")
    got = ops.linear_attention_fwd(q, k, x, sl, cu_seqlens=cu)[0]
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, 111:112, 2:, 7] = hit[0, 112:, :2, 5] = True
    assert torch.equal(got[~hit], out[~hit]) and not torch.isfinite(got[hit]).any()
    dq, dk, dv = ops.linear_attention_bwd(q, k, v, sl, d, cu_seqlens=cu)[:3]
    hit = torch.zeros_like(dq, dtype=torch.bool)
    hit[0, 44, 3] = hit[0, 45, 0] = True
    assert torch.equal(dq[~hit], grads[0][~hit]) and not torch.isfinite(dq[hit]).any()
    hit = torch.zeros_like(dv, dtype=torch.bool)
    hit[0, :45, 1, 9] = hit[0, 45, 0, 2] = True
    assert torch.equal(dv[~hit], grads[2][~hit]) and not torch.isfinite(dv[hit]).any()
    hit = torch.zeros_like(dk, dtype=torch.bool)
    hit[0, :45, 1] = hit[0, 45, 0] = True
    assert torch.equal(dk[~hit], grads[1][~hit]) and not torch.isfinite(dk[hit]).any()


# ------------------------------------------------------------------------------------------------ many sequences in one call
def test_workspace_of_a_packed_call_does_not_grow_with_its_sequences():
    """states are kept for segments that another one starts from: fewer than rows / segment, whatever the number of sequences"""
    from animal2vec_amd import _lib
    lib = _lib.load()
    for rows, H, HK, HD in ((400000, 16, 16, 64), (140000, 16, 16, 128), (5000, 2, 1, 32)):
        for back in (0, 1):
            size = lambda B: lib.a2v_linear_attention_workspace(1, back, 1, B, rows, H, HK, HD)        # noqa: E731
            own = size(1) - (2 * rows * H * HD * 4 if back and H != HK else 0)
            assert own <= (back + 1) * 1024 * HD * HD * 4                  # a state for each workgroup that fills the card
            assert all(size(B) == size(1) for B in (2, 100, 10000, 1000000))


def packed_reference(lens, q, k, v, slopes, scale, state, d_out, d_state):
    """ref_linear for packed rows in 64 bits, all sequences side by side"""
    T, H, D = q.shape
    rep, B, dev = H // k.shape[1], len(lens), q.device
    q, k, v, d_out = (t.double() for t in (q, k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1), d_out))
    n = torch.tensor(lens, device=dev)
    begin, end = n.cumsum(0) - n, n.cumsum(0)
    lam = torch.exp(-slopes.double())[:, None, None]
    st, g = state.double().clone(), d_state.double().clone()
    out, dq, dk, dv = (torch.zeros_like(q) for _ in range(4))
    for i in range(max(lens)):
        b = (n > i).nonzero()[:, 0]
        t = begin[b] + i
        st[b] = lam * st[b] + k[t].unsqueeze(-1) * v[t].unsqueeze(-2)
        out[t] = scale * (q[t].unsqueeze(-1) * st[b]).sum(-2)
        dq[t] = scale * (st[b] * d_out[t].unsqueeze(-2)).sum(-1)
        t = end[b] - 1 - i
        d = g[b] + scale * q[t].unsqueeze(-1) * d_out[t].unsqueeze(-2)
        dk[t] = (d * v[t].unsqueeze(-2)).sum(-1)
        dv[t] = (k[t].unsqueeze(-1) * d).sum(-2)
        g[b] = lam * d
    fold = lambda x: x.reshape(T, H // rep, rep, D).sum(2)      # noqa: E731
    return out, st, dq, fold(dk), fold(dv), g


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,HK,HD", [(2, 1, 32), (2, 2, 64)])
def test_many_packed_sequences(ops, dtype, H, HK, HD):
    """thousands of short and empty sequences around ones of exactly one, two, 17 and 18 segments (of 2 HD rows) and a row more or less: a
    neighbour's states are neither taken nor overwritten, and every sequence finds its rows"""
    seg, r = 2 * HD, torch.Generator().manual_seed(5)
    short = lambda n: torch.randint(0, 4, (n,), generator=r).tolist()         # noqa: E731
    lens = [0, 0, seg, seg, 2 * seg, 1, seg - 1, seg + 1, 3 * seg, 17 * seg, 18 * seg + 1] + short(1500) + [20 * seg - 7] + short(70) + [2 * seg + 5, 0, seg, 17 * seg + 1] + short(3000)
    T, B = sum(lens), len(lens)
    q, k, v, do = (rnd(1, T, h, HD, seed=i, dtype=dtype).cuda() for i, h in enumerate((H, HK, HK, H)))
    st, ds = rnd(B, H, HD, HD, seed=7, scale=2.0).cuda(), rnd(B, H, HD, HD, seed=8).cuda()
    sl = torch.tensor([0.002, 0.03], device="cuda")
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    got = (*ops.linear_attention_fwd(q, k, v, sl, state=st, want_state=True, cu_seqlens=cu),
           *ops.linear_attention_bwd(q, k, v, sl, do, state=st, d_state=ds, cu_seqlens=cu))
    want = packed_reference(lens, q[0], k[0], v[0], sl, HD ** -0.5, st, do[0], ds)
    size = packed_reference(lens, q[0].abs(), k[0].abs(), v[0].abs(), sl, HD ** -0.5, st.abs(), do[0].abs(), ds.abs())
    c = c_of(dtype, max(lens), HD)
    for g, w, m, name in zip(got, want, size, ("out", "last", "dq", "dk", "dv", "first")):
        check(g[0] if name not in ("last", "first") else g, w.cpu(), m.cpu(), c, name)


@gpu
def test_sequences_are_found_among_any_number(ops):
    """1, 2, 63 ... 70000 sequences, at the edges of what one, two and three looks of 64 lanes tell apart: sequence b's rows hold b + 1 and the
    state behind them says so"""
    H, HD = 1, 32
    for B in (1, 2, 63, 64, 65, 128, 4095, 4096, 4097, 4225, 70000):
        lens = torch.randint(0, 3, (B,), generator=torch.Generator().manual_seed(B))
        cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).to(torch.int32).cuda() + 3
        T = int(cu[-1]) + 200
        of = torch.repeat_interleave(torch.arange(1, B + 1), lens).float().cuda()
        k = torch.full((1, T, H, HD), 9.0, device="cuda")
        v = torch.zeros(1, T, H, HD, device="cuda")
        k[0, 3:T - 200], v[0, 3:T - 200, 0, 0] = 1.0, of
        out, last = ops.linear_attention_fwd(k, k, v, torch.zeros(H, device="cuda"), scale=1.0, cu_seqlens=cu, want_state=True)
        want = lens.cuda() * torch.arange(1, B + 1, device="cuda")         # (below 2^24: exact)
        assert torch.equal(last[:, 0, :, 0], want.float()[:, None].expand(B, HD)) and not last[:, 0, :, 1:].any(), B
        first = torch.cat([torch.ones(1, device="cuda"), (of[1:] != of[:-1]).float()]) if len(of) else of
        assert torch.equal(out[0, 3:T - 200, 0, 0], HD * of * (2 - first)), B
        assert not out[0, :3].any() and not out[0, T - 200:].any(), B


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,HK,HD,pool,shift", [(511, 3, 1, 32, 200, 1), (512, 2, 2, 64, 600, 0), (1100, 4, 2, 32, 300, 2), (1700, 4, 4, 64, 1500, 3), (3001, 4, 1, 32, 3500, 1), (5, 2, 1, 32, 3, 3)])
def test_step_of_many_rows(ops, N, H, HK, HD, pool, shift, dtype):
    """several heads to a workgroup (a number that need not divide them), slots that start anywhere, named once, often, or outside the pool"""
    r = torch.Generator().manual_seed(N)
    slots = torch.randint(-3, pool + 3, (N + shift,), generator=r, dtype=torch.int32)
    qkv = rnd(N, H + 2 * HK, HD, seed=1, dtype=dtype)
    state, sl, scale = rnd(pool, H, HD, HD, seed=2), alibi(H), HD ** -0.5
    sd, x = state.cuda(), qkv.cuda()
    out = ops.linear_attention_step(x[:, :H], x[:, H:H + HK], x[:, H + HK:], sl.cuda(), sd, slots=slots.cuda()[shift:])
    sel = slots[shift:].tolist()
    lam = torch.exp(-sl.double())[:, None, None]
    want, size = state.double(), state.double().abs()
    o, m = torch.zeros(N, H, HD, dtype=torch.float64), torch.zeros(N, H, HD, dtype=torch.float64)
    count = [0] * pool
    for n, s in enumerate(sel):
        if 0 <= s < pool:
            q, k, v = (t.double() for t in (qkv[n, :H], qkv[n, H:H + HK].repeat_interleave(H // HK, 0), qkv[n, H + HK:].repeat_interleave(H // HK, 0)))
            kv = k.unsqueeze(-1) * v.unsqueeze(-2)
            want[s], size[s] = lam * want[s] + kv, lam * size[s] + kv.abs()
            o[n], m[n] = scale * (q.unsqueeze(-1) * want[s]).sum(-2), scale * (q.abs().unsqueeze(-1) * size[s]).sum(-2)
            count[s] += 1
    c = (HD + 16 + 4 * max(count)) * 2.0 ** -24
    check(out, o, m, c, "out")
    check(sd, want, size, c, "states")
    assert not out[[n for n, s in enumerate(sel) if not 0 <= s < pool]].any()


# ------------------------------------------------------------------------------------------------ tensors that share a buffer
def test_overlap_is_what_the_elements_say():
    """small strided views of one buffer against their elements one by one"""
    import itertools
    import random
    from animal2vec_amd import ops
    r, buf, met = random.Random(1), torch.zeros(4000, dtype=torch.bfloat16), 0

    def view():
        dims = r.randint(2, 4)
        return buf.as_strided([r.randint(1, 4) for _ in range(dims)], [r.choice([0, 1, 2, 3, 5, 8, 12, 16, 24, 40, 64, 96, 200]) for _ in range(dims)], r.randint(0, 600))

    def elements(t):
        return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))}
    for _ in range(4000):
        a, b = view(), view()
        share = bool(elements(a) & elements(b))
        assert ops._overlap(a, b) == share, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        met += share
    assert 100 < met < 3900


PACKED = {"heads outermost": (lambda n, s, h, d: (n, s, h, 3, d), 3, (0, 1, 2, 3)), "slots outermost": (lambda n, s, h, d: (3, n, s, h, d), 0, (0, 1, 2, 3)),
          "rows innermost": (lambda n, s, h, d: (n, 3, h, s, d), 1, (0, 2, 1, 3)), "rows of heads": (lambda n, s, h, d: (n, h, 3, s, d), 2, (0, 2, 1, 3))}


def packed_slots(layout, N, S, H, HD, **kw):
    shape, dim, order = PACKED[layout]
    return [t.permute(order) for t in torch.zeros(*shape(N, S, H, HD), **kw).unbind(dim)]


@pytest.mark.parametrize("layout", PACKED)
def test_slots_of_any_packed_buffer_are_taken(layout):
    """results beside each other in one buffer, whichever dimension the slots lie between, reach the device check; a slot moved onto its
    neighbour does not"""
    from animal2vec_amd import _lib, ops
    N, S, H, HD = 2, 5, 4, 64
    q, k, v = packed_slots(layout, N, S, H, HD, dtype=torch.bfloat16)
    g = packed_slots(layout, N, S, H, HD, dtype=torch.bfloat16)
    w, f, sl, do = torch.zeros(HD), torch.zeros(HD // 2), torch.zeros(H), torch.zeros(N, S, H, HD, dtype=torch.bfloat16)
    for go in (lambda: ops.linear_attention_bwd(q, k, v, sl, do, dq=g[0], dk=g[1], dv=g[2]), lambda: ops.linear_attention_fwd(q, k, do, sl, out=v),
               lambda: ops.qk_norm_rope_fwd(q, k, w, w, f, q_out=q, k_out=k)):
        with pytest.raises(_lib.A2VError):
            go()
    onto = g[1].as_strided(g[1].shape, g[1].stride(), g[1].storage_offset() - HD // 2)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_attention_bwd(q, k, v, sl, do, dq=g[0], dk=onto, dv=g[2])


@gpu
@pytest.mark.parametrize("layout", PACKED)
def test_results_in_slots_of_any_packed_buffer(ops, layout):
    N, S, H, HD = 2, 75, 4, 64
    q, k, v = packed_slots(layout, N, S, H, HD, dtype=torch.bfloat16, device="cuda")
    for i, t in enumerate((q, k, v)):
        t.copy_(rnd(N, S, H, HD, seed=i))
    do, sl, w, f = rnd(N, S, H, HD, seed=4, dtype=torch.bfloat16).cuda(), alibi(H).cuda(), 1 + 0.1 * rnd(HD, seed=5).cuda(), ops.rope_inv_freq((HD // 2,))
    want = ops.linear_attention_bwd(q.contiguous(), k.contiguous(), v.contiguous(), sl, do)[:3]
    g = packed_slots(layout, N, S, H, HD, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        ops.linear_attention_bwd(q, k, v, sl, do, dq=g[0], dk=g[1], dv=g[2])
    assert all(torch.equal(a, b) for a, b in zip(g, want))
    want, kept = ops.qk_norm_rope_fwd(q.contiguous(), k.contiguous(), w, w, f), v.clone()
    ops.qk_norm_rope_fwd(q, k, w, w, f, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
