"""Timed cases of the operators around linear attention: norm and rotation of queries and keys, linear attention with a decay per
head in its chunked form (forward and training), and its recurrent form for single tokens.

The formulas, for one head of HD channels:

  norm and rotation   y = R(pos) (x / sqrt(mean(x^2) + eps) * w), R turning the pair of channels (a_i, b_i) by pos_axis(i) * inv_freq_i
  linear attention    S_t = exp(-slope) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t

`own` false: elementary torch operations in 32 bits, rounded once at the end.  `own` true: the calls of animal2vec_amd.ops.
"""
import math
import random

import torch

own = False

FRAMES = 200            # frames per second of the encoder (8 kHz clips, 40 samples per frame)
DAY = 24 * 3600 * FRAMES
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    rope = dict(op="norm_rope", train=False, dtype="bf16", n=1, s=1, heads=16, kv_heads=16, hd=64, rotary=64, axes=1, interleaved=False, first=0)
    lin = dict(op="linear", train=False, dtype="bf16", n=1, s=1, heads=16, kv_heads=16, hd=64, ragged=False, carry=False)
    step = dict(op="step", dtype="bf16", n=1, heads=16, kv_heads=16, hd=64, pool=0)
    return [
        # the teacher's view of a pretraining micro-batch: 64 clips of 10 s, every frame
        dict(rope, name="norm_rope_clips", n=64, s=2000),
        # the student's kept frames, forward and backward, with a position in time, microphone and band each
        dict(rope, name="norm_rope_train_kept", train=True, n=192, s=140, axes=3),
        # odd sizes in the parity mode: shared key heads, half of the channels turned, neighbouring channels as pairs
        dict(rope, name="norm_rope_odd_fp32", dtype="fp32", n=3, s=1021, heads=12, kv_heads=4, rotary=32, interleaved=True),
        # one frame each of five streams that have been running for a day, in the half-precision library
        dict(rope, name="norm_rope_frame", dtype="fp16", n=5, s=1, hd=128, rotary=128, heads=8, kv_heads=2, first=DAY),
        # the same micro-batch through the attention
        dict(lin, name="linear_clips", n=64, s=2000),
        # one recording of ten minutes: few rows, a long axis
        dict(lin, name="linear_recording", s=600 * FRAMES, carry=True),
        # clips of very different lengths in one call, continued from states, empty ones among them
        dict(lin, name="linear_ragged", n=37, s=6007, heads=12, kv_heads=4, ragged=True, carry=True),
        # training on the student's kept frames
        dict(lin, name="linear_train_kept", train=True, n=192, s=140),
        # training on 10 s at 44.1 kHz
        dict(lin, name="linear_train_long", train=True, n=4, s=11025),
        # training in the parity mode
        dict(lin, name="linear_train_fp32", train=True, dtype="fp32", n=2, s=2000, heads=12, kv_heads=12),
        # one frame of one stream
        dict(step, name="step_one"),
        # one frame each of 256 streams whose states live in a pool
        dict(step, name="step_pool", n=256, pool=320),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "linear", "linear", "linear", "step"])
    hd = rng.choice([32, 64, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 4]) if kv <= 4 else kv
    width = heads * hd / 1024
    if op == "step":
        n = _spread(rng, 1, max(2, min(256, int(200 * 64 / hd / width))))
        return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), n=n, heads=heads, kv_heads=kv, hd=hd, pool=rng.choice([0, n + rng.randint(1, 40)]))
    train = rng.random() < 0.5
    if op == "norm_rope":
        rows = _spread(rng, 1, 40000 / max(1.0, width))
        n = rng.choice([1, 2, 3, 5, 8, 13, 32])
        return dict(op=op, train=train, dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]), n=n, s=max(1, rows // n), heads=heads, kv_heads=kv, hd=hd,
                    rotary=rng.choice([hd, hd, hd // 2]), axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.5,
                    first=rng.choice([0, 0, rng.randint(1, 5 * DAY)]))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    rows = _spread(rng, 1, (30000 if dtype == "bf16" else 8000) / max(1.0, width) * min(1.0, 64 / hd) / (2 if train else 1))
    n = min(rows, rng.choice([1, 1, 2, 3, 8, 21, 64]))
    ragged = rng.random() < 0.4
    return dict(op=op, train=train, dtype=dtype, n=n, s=max(1, rows // n), heads=heads, kv_heads=kv, hd=hd, ragged=ragged, carry=rng.random() < 0.5)


def _lengths(c):
    """Rows of each sequence: all alike, or (ragged) spread over a factor of 100 with an empty one among them, n * s // 4 in all."""
    if not c["ragged"]:
        return [c["s"]] * c["n"]
    r = random.Random(c["n"] * 1000003 + c["s"])
    share = [math.exp(r.uniform(math.log(0.01), 0.0)) for _ in range(c["n"])]
    if c["n"] > 2:
        share[c["n"] // 2] = 0.0
    total = max(1, c["n"] * c["s"] // 4)
    got = [int(total * x / sum(share)) for x in share]
    got[0] += total - sum(got)
    return got


def _sections(c):
    half = c["rotary"] // 2
    small = half // 4
    return (half - small * (c["axes"] - 1),) + (small,) * (c["axes"] - 1)


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    hd, heads, kv = c["hd"], c["heads"], c["kv_heads"]
    if c["op"] == "step":
        return {"bytes": c["n"] * (heads * hd * hd * 8 + (2 * heads + 2 * kv) * hd * size), "flops": 5 * c["n"] * heads * hd * hd}
    if c["op"] == "norm_rope":
        rows = c["n"] * c["s"]
        one = rows * (heads + kv) * hd
        table = rows * 4 * c["axes"] + 8 * hd + 2 * c["rotary"]
        # training: x and y once, then x, dy and dx (the activations are far apart in time and pass through memory again)
        return {"bytes": one * size * (5 if c["train"] else 2) + table * (2 if c["train"] else 1), "flops": one * (24 if c["train"] else 8)}
    lens = _lengths(c)
    rows = sum(lens)
    fwd = rows * (2 * heads + 2 * kv) * hd * size
    states = c["n"] * heads * hd * hd * 4 * 2 if c["carry"] else 0
    bwd = rows * (3 * heads + 4 * kv) * hd * size
    return {"bytes": fwd + states + ((bwd + 2 * states) if c["train"] else 0), "flops": 4 * rows * heads * hd * hd * (4 if c["train"] else 1)}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    c = dict(case)
    dev = "cuda"
    g = torch.Generator(dev).manual_seed(int(seed))
    dt, hd, heads, kv = DTYPES[c["dtype"]], c["hd"], c["heads"], c["kv_heads"]

    def normal(*shape, dtype=dt, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    def unit(*shape):                     # what the norm leaves: rows of mean square 1
        x = torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)
        return (x * x.pow(2).mean(-1, keepdim=True).rsqrt()).to(dt)

    st = {"case": c}
    st["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device=dev, dtype=torch.float32) / heads)
    if c["op"] == "norm_rope":
        n, s = c["n"], c["s"]
        st["qkv"] = normal(n, s, (heads + 2 * kv), hd, scale=1.5)       # as the Linear wrote it: q, k and v of a row side by side
        st["wq"] = 1.0 + normal(hd, dtype=torch.float32, scale=0.2)
        st["wk"] = 1.0 + normal(hd, dtype=torch.float32, scale=0.2)
        st["sections"] = _sections(c)
        st["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(m, device=dev, dtype=torch.float64) / max(1, m)) for m in st["sections"]]).float()
        gaps = torch.randint(1, 15, (n, s), generator=g, device=dev)    # kept frames: ascending, with gaps
        time = (gaps.cumsum(1) - 1 + c["first"]).to(torch.int32)
        if c["axes"] == 1:
            st["pos"] = time
        else:
            rest = torch.randint(0, 64, (n, s, c["axes"] - 1), generator=g, device=dev, dtype=torch.int32)
            st["pos"] = torch.cat([time.unsqueeze(-1), rest], -1).contiguous()
        if c["train"]:
            st["dq"], st["dk"] = normal(n, s, heads, hd), normal(n, s, kv, hd)
        return st
    if c["op"] == "step":
        n, pool = c["n"], c["pool"] or c["n"]
        st["q"], st["k"], st["v"] = unit(n, heads, hd), unit(n, kv, hd), normal(n, kv, hd)
        st["state"] = normal(pool, heads, hd, hd, dtype=torch.float32, scale=3.0)
        st["slots"] = torch.randperm(pool, generator=g, device=dev)[:n].to(torch.int32) if c["pool"] else None
        return st
    lens = _lengths(c)
    n, s = (1, sum(lens)) if c["ragged"] else (c["n"], c["s"])
    st["q"], st["k"], st["v"] = unit(n, s, heads, hd), unit(n, s, kv, hd), normal(n, s, kv, hd)
    ends = torch.tensor([0] + lens, device=dev).cumsum(0)
    st["cu"] = ends.to(torch.int32) if c["ragged"] else None
    st["lens"] = lens
    st["state"] = normal(len(lens), heads, hd, hd, dtype=torch.float32, scale=3.0) if c["carry"] else None
    if c["train"]:
        st["d_out"] = normal(n, s, heads, hd)
        st["d_state"] = normal(len(lens), heads, hd, hd, dtype=torch.float32) if c["carry"] else None
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        from animal2vec_amd import ops
        if c["dtype"] == "fp16":
            with ops.half_library():
                return _own(ops, c, state)
        return _own(ops, c, state)
    if c["op"] == "norm_rope":
        return _plain_norm_rope(c, state)
    if c["op"] == "step":
        return _plain_step(c, state)
    return _plain_linear(c, state)


def _own(ops, c, t):
    if c["op"] == "norm_rope":
        q, k = t["qkv"][:, :, :c["heads"]], t["qkv"][:, :, c["heads"]:c["heads"] + c["kv_heads"]]
        how = dict(sections=t["sections"], interleaved=c["interleaved"], eps=1e-6)
        y = ops.qk_norm_rope_fwd(q, k, t["wq"], t["wk"], t["inv_freq"], t["pos"], **how)
        if not c["train"]:
            return y
        dwq, dwk = torch.zeros_like(t["wq"]), torch.zeros_like(t["wk"])
        dx = ops.qk_norm_rope_bwd(t["dq"], t["dk"], q, k, t["wq"], t["wk"], t["inv_freq"], t["pos"], dq_weight=dwq, dk_weight=dwk, **how)
        return (*y, *dx, dwq, dwk)
    if c["op"] == "step":
        out = ops.linear_attention_step(t["q"], t["k"], t["v"], t["slopes"], t["state"], slots=t["slots"])
        return out, t["state"]
    how = dict(state=t["state"], cu_seqlens=t["cu"])
    out, last = ops.linear_attention_fwd(t["q"], t["k"], t["v"], t["slopes"], want_state=c["carry"], **how)
    if not c["train"]:
        return out, last
    dq, dk, dv, first = ops.linear_attention_bwd(t["q"], t["k"], t["v"], t["slopes"], t["d_out"], d_state=t["d_state"], **how)
    return out, last, dq, dk, dv, first


# ------------------------------------------------------------------------------------------------ the plain forms
def _angles(c, t):
    """cos, sin (n, s, 1, rotary / 2) in 32 bits of angles formed in 64"""
    pos = t["pos"].unsqueeze(-1) if t["pos"].dim() == 2 else t["pos"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=pos.device), torch.tensor(t["sections"], device=pos.device),
                                   output_size=c["rotary"] // 2)
    a = pos.double()[..., axis] * t["inv_freq"].double()
    return a.cos().float().unsqueeze(2), a.sin().float().unsqueeze(2)


def _turn(c, x, cos, sin):
    r = c["rotary"]
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_norm_rope(c, t):
    dt = t["qkv"].dtype
    cos, sin = _angles(c, t)
    q, k = t["qkv"][:, :, :c["heads"]].float(), t["qkv"][:, :, c["heads"]:c["heads"] + c["kv_heads"]].float()
    rq, rk = (q.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt(), (k.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
    y = _turn(c, q * rq * t["wq"], cos, sin).to(dt), _turn(c, k * rk * t["wk"], cos, sin).to(dt)
    if not c["train"]:
        return y
    gq, gk = _turn(c, t["dq"].float(), cos, -sin), _turn(c, t["dk"].float(), cos, -sin)
    xq, xk = q * rq, k * rk
    dwq, dwk = (gq * xq).sum((0, 1, 2)), (gk * xk).sum((0, 1, 2))
    gq, gk = gq * t["wq"], gk * t["wk"]
    dq = rq * (gq - xq * (gq * xq).mean(-1, keepdim=True))
    dk = rk * (gk - xk * (gk * xk).mean(-1, keepdim=True))
    return (*y, dq.to(dt), dk.to(dt), dwq, dwk)


def _plain_step(c, t):
    rep = c["heads"] // c["kv_heads"]
    q, k, v = t["q"].float(), t["k"].float().repeat_interleave(rep, 1), t["v"].float().repeat_interleave(rep, 1)
    s = t["state"] if t["slots"] is None else t["state"][t["slots"].long()]
    s = s * torch.exp(-t["slopes"])[:, None, None] + k.unsqueeze(-1) * v.unsqueeze(-2)
    if t["slots"] is None:
        t["state"].copy_(s)
    else:
        t["state"][t["slots"].long()] = s
    out = (q.unsqueeze(-1) * s).sum(-2) * c["hd"] ** -0.5
    return out.to(t["q"].dtype), t["state"]


def _decays(slopes, n):
    """exp(-slope n), (heads, *n.shape), for whole numbers n; 0 where n < 0"""
    e = torch.exp(-slopes.double().reshape([-1] + [1] * n.dim()) * n.clamp(min=0).double())
    return torch.where(n >= 0, e, 0.0).float()


def _sums(q, k, v, slopes, first, lead):
    """sum_{j <= i} exp(-slope (i - j)) (q_i . k_j) v_j + exp(-slope (i + lead)) first^T q_i for q, k, v (b, heads, length, hd), in
    chunks: inside a chunk from the scores, from earlier chunks through the states at their ends."""
    b, h, length, d = q.shape
    size = 128
    n = -(-length // size)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * size - length)).reshape(b, h, n, size, d) for x in (q, k, v))
    i = torch.arange(size, device=q.device)
    c = torch.arange(n, device=q.device)
    scores = (q @ k.transpose(-1, -2).contiguous()) * _decays(slopes, i[:, None] - i[None, :])[:, None]
    ends = (k * _decays(slopes, size - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    start = _decays(slopes, (c[:, None] - 1 - c[None, :]) * size) @ ends.reshape(b, h, n, d * d)
    if first is not None:
        far = torch.exp(-slopes.double()[:, None] * (c * size + lead - 1).double()).float()
        start = start + far[..., None] * first.reshape(b, h, 1, d * d)
    out = scores @ v + (q * _decays(slopes, i + 1)[:, None, :, None]) @ start.reshape(b, h, n, d, d)
    return out.reshape(b, h, n * size, d)[:, :, :length]


def _last(k, v, slopes, first, lens):
    """exp(-slope len) first + sum_j exp(-slope (len - 1 - j)) k_j v_j^T: the state behind each sequence"""
    left = lens[:, None] - 1 - torch.arange(k.shape[2], device=k.device)[None, :]
    s = (k * _decays(slopes, left).transpose(0, 1).unsqueeze(-1)).transpose(-1, -2).contiguous() @ v
    return s if first is None else s + _decays(slopes, lens).transpose(0, 1)[..., None, None] * first


def _plain_linear(c, t):
    dt, h, kv, hd = t["q"].dtype, c["heads"], c["kv_heads"], c["hd"]
    rep, scale, slopes, dev = h // kv, hd ** -0.5, t["slopes"], t["q"].device
    n, longest = len(t["lens"]), max(t["lens"])
    cu = t["cu"].long() if c["ragged"] else torch.arange(n + 1, device=dev) * c["s"]
    lens = cu[1:] - cu[:-1]
    rows = t["q"].shape[0] * t["q"].shape[1]
    i = torch.arange(longest, device=dev)
    inside = (i[None, :] < lens[:, None])[:, None, :, None]
    there = (cu[:-1, None] + i[None, :]).clamp(max=rows - 1)
    back = (cu[1:, None] - 1 - i[None, :]).clamp(min=0)
    flat = torch.arange(rows, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), flat, right=True)
    at = flat - cu[seq]
    at_back = lens[seq] - 1 - at

    def pick(x, index):                   # packed rows -> (sequences, heads, length, hd), zeros behind each end
        x = x.reshape(rows, -1, hd)[index].float().transpose(1, 2)
        x = x.repeat_interleave(h // x.shape[1], 1)
        return torch.where(inside, x, 0.0)

    def pack(y, place, shared):
        y = y.transpose(1, 2)[seq, place]
        return (y.reshape(rows, kv, rep, hd).sum(2) if shared else y).to(dt).reshape(*t["q"].shape[:2], -1, hd)

    q, k, v = pick(t["q"], there), pick(t["k"], there), pick(t["v"], there)
    out = pack(_sums(q, k, v, slopes, t["state"], 1) * scale, at, False)
    last = _last(k, v, slopes, t["state"], lens) if c["carry"] else None
    if not c["train"]:
        return out, last
    do = pick(t["d_out"], there)
    turned = None if t["state"] is None else t["state"].transpose(-1, -2).contiguous()
    dq = pack(_sums(do, v, k, slopes, turned, 1) * scale, at, False)
    first = None
    if c["carry"]:
        rise = _decays(slopes, torch.where(i[None, :] < lens[:, None], i[None, :] + 1, -1)).transpose(0, 1)
        first = (q * rise.unsqueeze(-1)).transpose(-1, -2).contiguous() @ do * scale + _decays(slopes, lens).transpose(0, 1)[..., None, None] * t["d_state"]
    q, k, v, do = pick(t["q"], back), pick(t["k"], back), pick(t["v"], back), pick(t["d_out"], back)
    end = t["d_state"]
    dv = pack(_sums(k, q, do * scale, slopes, end, 0), at_back, True)
    dk = pack(_sums(v, do * scale, q, slopes, None if end is None else end.transpose(-1, -2).contiguous(), 0), at_back, True)
    return out, last, dq, dk, dv, first


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    c, t = case, prepare(case, seed)
    if c["op"] == "norm_rope":
        pos = t["pos"].reshape(c["n"], c["s"], c["axes"]).double()
        parts, at = [], 0
        for a, m in enumerate(t["sections"]):
            parts.append(pos[..., a, None] * t["inv_freq"][at:at + m].double())
            at += m
        angle = torch.cat(parts, -1).unsqueeze(2)
        spin = torch.polar(torch.ones_like(angle), angle)
        half, r = c["rotary"] // 2, c["rotary"]
        order = torch.arange(r, device=angle.device)
        order = order.reshape(half, 2) if c["interleaved"] else order.reshape(2, half).t()

        def turn(x, by):
            z = torch.complex(x[..., order[:, 0]], x[..., order[:, 1]]) * by
            y = x.clone()
            y[..., order[:, 0]], y[..., order[:, 1]] = z.real, z.imag
            return y

        got, grads, sums = [], [], []
        for x, w, d in ((t["qkv"][:, :, :c["heads"]], t["wq"], "dq"), (t["qkv"][:, :, c["heads"]:c["heads"] + c["kv_heads"]], t["wk"], "dk")):
            x, w = x.double(), w.double()
            length = (x.square().sum(-1, keepdim=True) / c["hd"] + 1e-6).sqrt()
            got.append(turn(x / length * w, spin))
            if c["train"]:
                back = turn(t[d].double(), spin.conj())
                sums.append((back * x / length).sum((0, 1, 2)))
                back = back * w
                grads.append(back / length - x * (back * x).sum(-1, keepdim=True) / (c["hd"] * length ** 3))
        return tuple(got) if not c["train"] else (*got, *grads, *sums)

    rep, scale = c["heads"] // c["kv_heads"], c["hd"] ** -0.5
    fade = torch.exp(-t["slopes"].double())[:, None, None]
    if c["op"] == "step":
        s, which = t["state"].double(), (t["slots"].long() if c["pool"] else torch.arange(c["n"], device=fade.device))
        k, v = t["k"].double().repeat_interleave(rep, 1), t["v"].double().repeat_interleave(rep, 1)
        s[which] = s[which] * fade + torch.einsum("nhi,nhj->nhij", k, v)
        return torch.einsum("nhi,nhij->nhj", t["q"].double(), s[which]) * scale, s

    lens = t["lens"]
    if max(lens) * (3 if c["train"] else 1) > 400_000:
        return None
    order = sorted(range(len(lens)), key=lambda b: -lens[b])            # longest first: the running ones stay in front
    starts = [sum(lens[:b]) for b in range(len(lens))]
    hd, h = c["hd"], c["heads"]
    flat = {x: t[x].reshape(-1, t[x].shape[-2], hd) for x in ("q", "k", "v", "d_out") if x in t and t[x] is not None}
    begin = torch.tensor([starts[b] for b in order], device=fade.device)
    size = torch.tensor([lens[b] for b in order], device=fade.device)
    live = [sum(1 for b in order if lens[b] > i) for i in range(max(lens))]
    zero = torch.zeros(len(lens), h, hd, hd, dtype=torch.float64, device=fade.device)
    out = torch.zeros(flat["q"].shape, dtype=torch.float64, device=fade.device)

    def row(x, at):
        x = flat[x][at].double()
        return x.repeat_interleave(h // x.shape[1], 1)

    s = t["state"].double()[order] if t["state"] is not None else zero.clone()
    grads = {x: torch.zeros(flat[x].shape[0], h, hd, dtype=torch.float64, device=fade.device) for x in ("q", "k", "v")} if c["train"] else {}
    for i, m in enumerate(live):
        at = begin[:m] + i
        q, k, v = row("q", at), row("k", at), row("v", at)
        s[:m].mul_(fade).add_(k.unsqueeze(-1) * v.unsqueeze(-2))
        out[at] = (q.unsqueeze(-2) @ s[:m]).squeeze(-2) * scale
        if c["train"]:
            grads["q"][at] = (s[:m] @ row("d_out", at).unsqueeze(-1)).squeeze(-1) * scale
    undo = sorted(range(len(lens)), key=lambda p: order[p])
    last = s[undo] if c["carry"] else None
    shape = t["q"].shape
    if not c["train"]:
        return out.reshape(shape), last
    g = t["d_state"].double()[order] if t["d_state"] is not None else zero.clone()
    for i, m in enumerate(live):
        at = begin[:m] + size[:m] - 1 - i
        q, k, v, do = row("q", at), row("k", at), row("v", at), row("d_out", at)
        g[:m].add_(q.unsqueeze(-1) * do.unsqueeze(-2), alpha=scale)
        grads["k"][at] = (g[:m] @ v.unsqueeze(-1)).squeeze(-1)
        grads["v"][at] = (k.unsqueeze(-2) @ g[:m]).squeeze(-2)
        g[:m].mul_(fade)
    first = g[undo] if c["carry"] else None
    dk, dv = (grads[x].reshape(-1, c["kv_heads"], rep, hd).sum(2).reshape(t[x].shape) for x in ("k", "v"))
    return out.reshape(shape), last, grads["q"].reshape(shape), dk, dv, first
