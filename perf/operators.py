"""What is measured of the attention operators: cases over their real range,
their plain form in elementary torch operations, and their definition in 64
bits.

  cross_attention   queries read an encoder's states of another length
                    (kernels.cross_attention), forward, backward, one token
  qk_norm_rope      RMS norm of each head of the queries and keys with the
                    position rotation in the same pass (kernels.qk_norm_rope)
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BASE = 10000.0


def _attn(name, dtype, b, tq, tk, h, hk, d, grad, kv_lens=False, q_lens=False, mask=False):
    return {"name": name, "op": "cross_attention", "dtype": dtype, "b": b, "tq": tq, "tk": tk,
            "h": h, "hk": hk, "d": d, "grad": grad, "kv_lens": kv_lens, "q_lens": q_lens,
            "mask": mask}


def _norm(name, dtype, b, tq, tk, h, hk, d, grad, rot, axes=1, interleaved=False, start=0):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "b": b, "tq": tq, "tk": tk,
            "h": h, "hk": hk, "d": d, "grad": grad, "rot": rot, "axes": axes,
            "interleaved": interleaved, "start": start}


def listed():
    return [
        # one new token of one sample against one caption: the latency of a call
        _attn("token, one caption", "bf16", 1, 1, 62, 4, 4, 64, False),
        # serving: one token each of a batch against long encoder states of
        # ragged lengths, four query heads to a key head: bound by reading K, V
        _attn("token, long states", "bf16", 16, 1, 8192, 32, 8, 128, False, kv_lens=True),
        # a handful of tokens against one long clip, some of its states masked
        _attn("few tokens, masked", "fp16", 4, 5, 1500, 12, 12, 64, False, mask=True),
        # training: 14 x 14 face regions read captions of ragged lengths
        _attn("regions read captions", "bf16", 64, 196, 32, 4, 4, 64, True, kv_lens=True),
        # training in full precision: words of ragged captions read the
        # regions, one head over the whole feature
        _attn("words read regions", "fp32", 64, 30, 196, 1, 1, 256, True, q_lens=True),
        # training, odd everything: head size, lengths, a mask, shared heads
        _attn("odd sizes, masked", "fp16", 3, 333, 777, 6, 3, 80, True, mask=True),
        # training on long states, as a decoder over an encoder does
        _attn("long states, training", "bf16", 4, 1024, 1500, 16, 4, 128, True, kv_lens=True),
        # the largest: a long prompt reads long states: bound by the matrix units
        _attn("long prompt", "bf16", 4, 2048, 4096, 16, 4, 128, False),
        # one new token far down its sequence
        _norm("token, far position", "bf16", 8, 1, 1, 32, 8, 128, False, 128, start=1000003),
        # training in full precision on the 14 x 14 grid (two position axes)
        _norm("region grid, training", "fp32", 64, 196, 196, 4, 4, 64, True, 64, axes=2),
        # a long prompt: one read and one write of everything
        _norm("long prompt, norm", "bf16", 4, 4096, 4096, 32, 8, 128, False, 128),
        # training on long sequences, half of each head rotated, pairs adjacent
        _norm("long sequence, training", "bf16", 2, 4096, 4096, 32, 8, 128, True, 64,
              interleaved=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {}
    for c in listed():
        k = (c["op"], c["grad"])
        most[k] = max(most.get(k, 0), _cost(c))
    while True:
        grad = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 1, 2, 4])
        if rng.random() < 0.6:
            d = rng.choice([32, 36, 64, 64, 80, 96, 128, 128, 200, 256])
            form = "rows" if grad else rng.choice(["token", "few", "rows"])
            tq = 1 if form == "token" else _log_int(rng, 2, 16) if form == "few" else \
                _log_int(rng, 17, 2048)
            tk = _log_int(rng, 16, 8192)
            c = _attn("", dtype, _log_int(rng, 1, 64), tq, tk, h, hk, d, grad,
                      kv_lens=rng.random() < 0.5, q_lens=tq > 1 and rng.random() < 0.3,
                      mask=rng.random() < 0.3)
            # the score matrix of the plain form stays within a few GB
            if c["b"] * c["h"] * c["tq"] * c["tk"] > 4 * 16 * 2048 * 4096:
                continue
        else:
            d = rng.choice([32, 36, 64, 64, 80, 128, 128, 256])
            t = _log_int(rng, 1, 4096)
            axes = rng.choice([1, 1, 2]) if d % 4 == 0 else 1
            rot = d if rng.random() < 0.6 else d // 2 // (2 * axes) * (2 * axes)
            c = _norm("", dtype, _log_int(rng, 1, 64), t, _log_int(rng, 1, 4096), h, hk, d, grad,
                      rot, axes, rng.random() < 0.4, rng.choice([0, 17, 100000]))
        if _cost(c) <= most[(c["op"], c["grad"])]:
            del c["name"]
            return c


def work(case):
    """Each input read once and each output written once; the products that
    the formulas cannot do without (two forward, five more backward), over
    whole lengths."""
    c, s = case, DTYPES[case["dtype"]].itemsize
    nq, nk = c["b"] * c["tq"] * c["h"] * c["d"], c["b"] * c["tk"] * c["hk"] * c["d"]
    if c["op"] == "cross_attention":
        prod = 2 * c["b"] * c["h"] * c["tq"] * c["tk"] * c["d"]
        # forward: q, k, v -> o; backward: do -> dq, dk, dv
        return {"bytes": s * (2 * nq + 2 * nk + (2 * nq + 2 * nk if c["grad"] else 0)),
                "flops": prod * (7 if c["grad"] else 2)}
    n = nq + nk
    return {"bytes": s * n * (4 if c["grad"] else 2), "flops": n * (30 if c["grad"] else 10)}


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _positions(c, t):
    if c["axes"] == 1:
        return (c["start"] + torch.arange(t, device="cuda")).expand(c["b"], t).contiguous()
    w = max(1, math.isqrt(t))
    i = torch.arange(t, device="cuda")
    return torch.stack([c["start"] + i // w, c["start"] + i % w], -1).expand(
        c["b"], t, 2).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    q = _randn(g, c["b"], c["tq"], c["h"], c["d"], dtype=dt)
    k = _randn(g, c["b"], c["tk"], c["hk"], c["d"], dtype=dt)
    s = {"case": dict(c), "q": q, "k": k}
    leaves = [q, k]
    if c["op"] == "cross_attention":
        s["v"] = _randn(g, c["b"], c["tk"], c["hk"], c["d"], dtype=dt)
        leaves.append(s["v"])

        def lens(t):
            n = torch.randint(max(1, t // 4), t + 1, (c["b"],), generator=g, device="cuda")
            n[0] = t
            return n.to(torch.int32)
        s["kv_lens"] = lens(c["tk"]) if c["kv_lens"] else None
        s["q_lens"] = lens(c["tq"]) if c["q_lens"] else None
        # true: this state is attended to
        s["mask"] = torch.rand(c["b"], c["tk"], generator=g, device="cuda") > 0.15 \
            if c["mask"] else None
        s["scale"] = 1.0 / math.sqrt(c["d"])
        if c["grad"]:
            s["do"] = _randn(g, c["b"], c["tq"], c["h"], c["d"], dtype=dt)
    else:
        s["wq"] = 1.0 + 0.2 * torch.randn(c["d"], generator=g, device="cuda")
        s["wk"] = 1.0 + 0.2 * torch.randn(c["d"], generator=g, device="cuda")
        leaves += [s["wq"], s["wk"]]
        s["q_pos"], s["k_pos"] = _positions(c, c["tq"]), _positions(c, c["tk"])
        if c["grad"]:
            s["dq"] = _randn(g, *q.shape, dtype=dt)
            s["dk"] = _randn(g, *k.shape, dtype=dt)
        if own:
            from text_guided_face_recognition_amd import kernels as K
            s["rope"] = K.Rope(c["rot"], base=BASE, axes=c["axes"],
                               interleaved=c["interleaved"], device="cuda")
    if c["grad"]:
        for x in leaves:
            x.requires_grad_()
    return s


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_attention(state) if state["case"]["op"] == "cross_attention" else \
            _plain_norm(state)


def _run_own(s):
    from text_guided_face_recognition_amd import kernels as K
    c = s["case"]
    if c["op"] == "cross_attention":
        o = K.cross_attention(s["q"], s["k"], s["v"], scale=s["scale"], q_lens=s["q_lens"],
                              kv_lens=s["kv_lens"], mask=s["mask"])
        if not c["grad"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    yq, yk = K.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], eps=EPS, rope=s["rope"],
                            q_pos=s["q_pos"], k_pos=s["k_pos"])
    if not c["grad"]:
        return {"q": yq, "k": yk}
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), (s["q"], s["k"], s["wq"], s["wk"]),
                                           (s["dq"], s["dk"]))
    return {"q": yq.detach(), "k": yk.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


# ------------------------------------------------------------- plain form ---
def _plain_attention(s):
    c, dt = s["case"], s["q"].dtype
    b, tq, tk, h, hk, d = (c[n] for n in ("b", "tq", "tk", "h", "hk", "d"))

    def rows(x):        # [B, Tq, H, D] -> [B, Hk, H/Hk * Tq, D]
        return x.float().view(b, tq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)

    def back(x):        # its inverse
        return x.view(b, hk, h // hk, tq, d).permute(0, 3, 1, 2, 4).reshape(b, tq, h, d)

    q = rows(s["q"])
    k, v = (s[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]             # [B, Hk, rows, Tk]
    keep = torch.ones(b, 1, 1, tk, dtype=torch.bool, device=q.device)
    if s["kv_lens"] is not None:
        keep = keep & (torch.arange(tk, device=q.device) < s["kv_lens"].view(b, 1, 1, 1))
    if s["mask"] is not None:
        keep = keep & s["mask"].view(b, 1, 1, tk)
    if s["q_lens"] is not None:
        live = torch.arange(tq, device=q.device) < s["q_lens"].view(b, 1)
        keep = keep & live.repeat(1, h // hk).view(b, 1, -1, 1)
    score = torch.where(keep, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    z = e.sum(-1, keepdim=True)
    p = e / torch.where(z == 0, 1.0, z)
    o = torch.matmul(p, v)
    out = {"o": back(o).to(dt)}
    if c["grad"]:
        do = rows(s["do"])
        dp = torch.matmul(do, v.transpose(2, 3))
        ds = p * (dp - (do * o).sum(-1, keepdim=True)) * s["scale"]
        out["dq"] = back(torch.matmul(ds, k)).to(dt)
        out["dk"] = torch.matmul(ds.transpose(2, 3), q).permute(0, 2, 1, 3).contiguous().to(dt)
        out["dv"] = torch.matmul(p.transpose(2, 3), do).permute(0, 2, 1, 3).contiguous().to(dt)
    return out


def _angles(c, pos):
    """cos and sin [B, T, 1, rot / 2], the angles formed in 64 bits."""
    per = c["rot"] // 2 // c["axes"]
    freq = BASE ** (-torch.arange(per, dtype=torch.float64, device=pos.device) / per)
    a = pos.double().view(c["b"], -1, c["axes"], 1) * freq
    a = a.reshape(c["b"], -1, 1, c["rot"] // 2)
    return torch.cos(a).float(), torch.sin(a).float()


def _rotated(c, u, cos, sin):
    r = c["rot"]
    if c["interleaved"]:
        a, b = u[..., 0:r:2], u[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = u[..., :r // 2], u[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, u[..., r:]], -1)


def _plain_norm(s):
    c, out = s["case"], {}
    for n in ("q", "k"):
        x, w = s[n].float(), s["w" + n].float()
        cos, sin = _angles(c, s[n + "_pos"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        unit = x * r
        out[n] = _rotated(c, unit * w, cos, sin).to(s[n].dtype)
        if c["grad"]:
            du = _rotated(c, s["d" + n].float(), cos, -sin)
            out["dw" + n] = (du * unit).sum((0, 1, 2))
            du = du * w
            out["d" + n] = (r * (du - unit * (du * unit).mean(-1, keepdim=True))).to(s[n].dtype)
    return out


# ------------------------------------------------------------- definition ---
def exact(case, seed):
    c, s = case, prepare(case, seed)
    return _exact_attention(c, s) if c["op"] == "cross_attention" else _exact_norm(c, s)


def _exact_attention(c, s):
    """Sample by sample over the states that are attended to alone, with
    softmax and its derivative from torch in 64 bits."""
    q, k, v = (s[n].detach().double().requires_grad_(c["grad"]) for n in ("q", "k", "v"))
    o = torch.zeros_like(q.detach())
    grads = [torch.zeros_like(x.detach()) for x in (q, k, v)]
    for b in range(c["b"]):
        nq = c["tq"] if s["q_lens"] is None else int(s["q_lens"][b])
        nk = c["tk"] if s["kv_lens"] is None else int(s["kv_lens"][b])
        at = torch.arange(nk, device=q.device)
        if s["mask"] is not None:
            at = at[s["mask"][b, :nk]]
        if not nq or not at.numel():
            continue
        share = c["h"] // c["hk"]
        qb = q[b, :nq].transpose(0, 1)
        kb, vb = (x[b, at].transpose(0, 1).repeat_interleave(share, 0) for x in (k, v))
        ob = torch.softmax(qb @ kb.transpose(1, 2) * s["scale"], -1) @ vb
        o[b, :nq] = ob.detach().transpose(0, 1)
        if c["grad"]:
            got = torch.autograd.grad(ob.transpose(0, 1), (q, k, v), s["do"][b, :nq].double())
            for total, x in zip(grads, got):
                total[b] += x[b]
    out = {"o": o}
    if c["grad"]:
        out.update(zip(("dq", "dk", "dv"), grads))
    return out


def _exact_norm(c, s):
    """The pairs as complex numbers, turned by exp(i angle), in 64 bits."""
    out = {}
    half, per = c["rot"] // 2, c["rot"] // 2 // c["axes"]
    pair = torch.arange(half, device="cuda")
    axis, step = pair // per, (pair % per).double()
    for n in ("q", "k"):
        x = s[n].detach().double().requires_grad_(c["grad"])
        w = s["w" + n].detach().double().requires_grad_(c["grad"])
        pos = s[n + "_pos"].double().view(c["b"], -1, c["axes"])[..., axis]
        turn = torch.polar(torch.ones_like(pos), pos * torch.pow(BASE, -step / per)).unsqueeze(2)
        u = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if c["interleaved"]:
            z = torch.view_as_complex(u[..., :c["rot"]].unflatten(-1, (half, 2)).contiguous())
            y = torch.view_as_real(z * turn).flatten(-2)
        else:
            z = torch.complex(u[..., :half], u[..., half:c["rot"]]) * turn
            y = torch.cat([z.real, z.imag], -1)
        y = torch.cat([y, u[..., c["rot"]:]], -1)
        out[n] = y.detach()
        if c["grad"]:
            out["d" + n], out["dw" + n] = torch.autograd.grad(y, (x, w), s["d" + n].double())
    return out
