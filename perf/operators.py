"""The operators of a gated recurrent block, each as one pass that a program of this package makes.

``gated_recurrence`` is a linear recurrence with a matrix state per head and one decay per head and
step, trained on batches of windows and run over whole recordings; ``gated_recurrence_step`` is its
form for one token with the state carried; ``gated_norm`` is the norm with a gate behind it;
``residual_norm`` is the post-norm, residual scale, residual sum and the next block's pre-norm
between two blocks. With ``own`` the calls are the package's; without, the same operators in
elementary torch operations in float32. ``exact`` is the definition in float64, step by step.

Widths and lengths are those of the package's benchmark (batch 16, length 4096, width 1536) and of
identification models (windows of 512, narrow heads), with the odd sizes such models come to.
"""

from __future__ import annotations

import math

import torch

own = False

_IO = {"fp32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


def listed():
    return [
        # one sample of one model running on-line, in a control loop
        dict(name="step_online", kind="step", B=1, H=4, Hk=4, K=64, V=64, io="fp32"),
        # one token for each of a batch of served sequences, at the benchmark's width
        dict(name="step_serving", kind="step", B=256, H=12, Hk=12, K=128, V=128, io="bf16"),
        # prediction over whole recordings with the state carried in, few rows and a long time axis
        dict(name="recurrence_recording", kind="predict", B=1, L=65536, H=6, Hk=6, K=64, V=64, io="bf16", state=True, reset=False),
        # the first window of a session: a short prompt before the steps
        dict(name="recurrence_prompt", kind="predict", B=1, L=77, H=4, Hk=4, K=64, V=64, io="fp32", state=False, reset=False),
        # a training step on a batch of windows, an identification model's width
        dict(name="recurrence_windows", kind="train", B=64, L=512, H=2, Hk=2, K=64, V=64, io="fp32", state=True, reset=False),
        # a training step at the benchmark's batch, length and width
        dict(name="recurrence_large", kind="train", B=16, L=4096, H=12, Hk=12, K=128, V=128, io="bf16", state=False, reset=False),
        # windows of several recordings packed into rows (a decay of zero where one begins), queries and keys shared by heads
        dict(name="recurrence_packed", kind="train", B=5, L=3001, H=6, Hk=2, K=48, V=80, io="bf16", state=False, reset=True),
        # the norm with its gate behind one token of one sequence
        dict(name="gated_norm_token", kind="gnorm", rows=1, D=1536, groups=12, io="bf16", first=False, train=False),
        # the same behind the recurrence of the large training step, one group per head
        dict(name="gated_norm_large", kind="gnorm", rows=65536, D=1536, groups=12, io="bf16", first=False, train=True),
        # gate before the norm, over a narrow model's whole rows of odd width
        dict(name="gated_norm_odd", kind="gnorm", rows=32000, D=195, groups=1, io="fp32", first=True, train=True),
        # between two blocks, one token for each of a few sequences
        dict(name="residual_norm_tokens", kind="rnorm", rows=8, D=1536, io="bf16", res="fp32", post=True, scale=True, train=False),
        # between two blocks of the large training step
        dict(name="residual_norm_large", kind="rnorm", rows=65536, D=1536, io="bf16", res="bf16", post=True, scale=True, train=True),
    ]


# ---------------------------------------------------------------------------------- drawn sizes


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng, most):
    group = rng.choice([1, 1, 1, 2, 3])
    Hk = _log(rng, 1, max(1, most // group))
    return Hk * group, Hk


def _width(rng):
    return rng.choice([16, 24, 32, 48, 64, 64, 80, 96, 100, 128, 128, rng.randint(8, 128)])


def _draw_once(rng):
    kind = rng.choice(["step", "step", "predict", "predict", "train", "train", "train", "gnorm", "gnorm", "rnorm", "rnorm"])
    io = rng.choice(["fp32", "bf16"])
    if kind == "step":
        H, Hk = _heads(rng, 24)
        return dict(kind=kind, B=_log(rng, 1, 256), H=H, Hk=Hk, K=_width(rng), V=_width(rng), io=io)
    if kind == "predict":
        H, Hk = _heads(rng, 16)
        return dict(kind=kind, B=_log(rng, 1, 16), L=_log(rng, 20, 65536), H=H, Hk=Hk, K=_width(rng), V=_width(rng), io=io,
                    state=rng.random() < 0.5, reset=rng.random() < 0.3)
    if kind == "train":
        H, Hk = _heads(rng, 16)
        return dict(kind=kind, B=_log(rng, 1, 64), L=_log(rng, 100, 8192), H=H, Hk=Hk, K=_width(rng), V=_width(rng), io=io,
                    state=rng.random() < 0.4, reset=rng.random() < 0.3)
    train = rng.random() < 0.6
    rows = _log(rng, 200, 65536) if train else _log(rng, 1, 2048)
    if kind == "gnorm":
        groups = rng.choice([1, 1, 2, 4, 12])
        return dict(kind=kind, rows=rows, D=groups * _log(rng, 16, max(17, 2048 // groups)), groups=groups, io=io,
                    first=rng.random() < 0.4, train=train)
    return dict(kind=kind, rows=rows, D=_log(rng, 64, 2048), io=io, res=rng.choice([io, "fp32"]), post=rng.random() < 0.7,
                scale=rng.random() < 0.7, train=train)


def _size(case):
    """A rough cost of one pass: the inputs' elements, and the products between steps of a chunk for fp32 ones."""
    if case["kind"] == "step":
        return case["B"] * case["H"] * case["K"] * case["V"] / (256 * 12 * 128 * 128)
    if case["kind"] in ("gnorm", "rnorm"):
        return case["rows"] * case["D"] / (65536 * 1536)
    both = case["B"] * case["L"] * case["H"] * (64 + case["K"] + case["V"]) / (16 * 4096 * 12 * (64 + 128 + 128))
    return both * (1.0 if case["kind"] == "train" else 0.4)


def draw(rng):
    while True:
        case = _draw_once(rng)
        if _size(case) <= 1.0 and case.get("L", 1) * case.get("B", 1) * case.get("H", 1) <= 16 * 4096 * 12:
            return case


# ------------------------------------------------------------------------------------- inputs


class _Inputs:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda").to(dtype)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda") * (hi - lo) + lo


def _decay(r, B, L, H, dtype, reset):
    """Log decays of a trained gate: heads that remember from a few to about a thousand steps, each
    step's a softplus of a normal; where rows are packed, -inf about every 300 steps."""
    rate = torch.exp(r.uniform(math.log(1e-3), math.log(0.3), H))
    g = -rate * torch.nn.functional.softplus(r.normal(B, L, H))
    if reset:
        starts = (r.uniform(0, 1, B, L) < 1 / 300)[..., None]
        g = g.masked_fill(starts, float("-inf"))
    return g.to(dtype)


def prepare(case, seed):
    r, c, kind = _Inputs(seed), case, case["kind"]
    dt = _IO[case["io"]]
    s = dict(case=dict(case))
    if kind == "step":
        B, H, Hk, K, V = (c[n] for n in ("B", "H", "Hk", "K", "V"))
        s.update(q=r.normal(B, Hk, K, dtype=dt), k=(r.normal(B, Hk, K) / math.sqrt(K)).to(dt), v=r.normal(B, H, V, dtype=dt),
                 g=_decay(r, B, 1, H, dt, False)[:, 0], state=r.normal(B, H, K, V))
    elif kind in ("predict", "train"):
        B, L, H, Hk, K, V = (c[n] for n in ("B", "L", "H", "Hk", "K", "V"))
        s.update(q=r.normal(B, L, Hk, K, dtype=dt), k=(r.normal(B, L, Hk, K) / math.sqrt(K)).to(dt), v=r.normal(B, L, H, V, dtype=dt),
                 g=_decay(r, B, L, H, dt, c["reset"]), state=r.normal(B, H, K, V) if c["state"] else None)
        if kind == "train":
            s.update(do=r.normal(B, L, H, V, dtype=dt), dstate=r.normal(B, H, K, V) if c["state"] else None)
            s["leaves"] = [s[n].requires_grad_() for n in ("q", "k", "v", "g", "state") if s[n] is not None]
    else:
        rows, D = c["rows"], c["D"]
        s.update(x=r.normal(rows, D, dtype=dt), w=r.uniform(0.5, 1.5, D))
        names = ["x"]
        if kind == "gnorm":
            s["gate"] = r.normal(rows, D, dtype=dt)
            names += ["gate", "w"]
        else:
            s["r"] = r.normal(rows, D, dtype=_IO[c["res"]])
            s["wpost"] = r.uniform(0.5, 1.5, D) if c["post"] else None
            s["scale"] = r.uniform(0.05, 0.5, D) if c["scale"] else None
            names += ["r", "w", "wpost", "scale"]
        if c["train"]:
            s["dy"] = r.normal(rows, D, dtype=dt)
            if kind == "rnorm":
                s["dr"] = r.normal(rows, D, dtype=_IO[c["res"]])
            s["leaves"] = [s[n].requires_grad_() for n in names if s[n] is not None]
    return s


# ----------------------------------------------------------------------------------- the passes


def _span_sums(g):
    """``[..., i, j]``: the sum of ``g`` over the steps after j up to i (0 at i = j, -inf above)."""
    n = g.shape[-1]
    at = torch.arange(n, device=g.device)
    below = at[:, None] > at
    sums = torch.where(below, g[..., :, None], 0.0).cumsum(-2)
    return sums.masked_fill(at[:, None] < at, float("-inf"))


def _plain_recurrence(q, k, v, g, state):
    B, L, H, V = v.shape
    K = q.shape[-1]
    C = 64 if L <= 8192 else 256
    n = -(-L // C)

    def chunks(t, heads):  # [B, heads, n, C, width]
        t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, n * C - L))
        return t.repeat_interleave(H // heads, 2).reshape(B, n, C, H, -1).permute(0, 3, 1, 2, 4)

    qc, kc, vc = chunks(q, q.shape[2]), chunks(k, k.shape[2]), chunks(v, H)
    gc = chunks(g[..., None], H)[..., 0]
    decay = _span_sums(gc).exp()  # [B, H, n, C, C]
    own_states = (kc * decay[..., -1, :, None]).transpose(-1, -2) @ vc  # [B, H, n, K, V]
    first = torch.zeros(B, H, K, V, device=v.device) if state is None else state
    between = _span_sums(torch.nn.functional.pad(gc.sum(-1), (1, 0))).exp()  # [B, H, n + 1, n + 1]
    states = between @ torch.cat((first[:, :, None], own_states), 2).flatten(-2)
    states = states.unflatten(-1, (K, V))
    o = (qc @ kc.transpose(-1, -2) * decay) @ vc + (qc * gc.cumsum(-1).exp()[..., None]) @ states[:, :, :-1]
    o = o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, V)[:, :L]
    return o.to(v.dtype), states[:, :, -1]


def _plain_step(q, k, v, g, state):
    group = v.shape[1] // q.shape[1]
    q, k = (t.float().repeat_interleave(group, 1) for t in (q, k))
    new = g.float().exp()[..., None, None] * state + k[..., None] * v.float()[..., None, :]
    state.copy_(new)
    return (q[..., None] * new).sum(-2).to(v.dtype)


def _rms(x, groups=1):
    x = x.unflatten(-1, (groups, -1))
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)).flatten(-2)


def _plain_gated_norm(x, gate, w, groups, first):
    x32, gate = x.float(), gate.float()
    act = gate * torch.sigmoid(gate)
    y = _rms(x32 * act, groups) * w if first else _rms(x32, groups) * w * act
    return y.to(x.dtype)


def _plain_residual_norm(x, r, w, wpost, scale):
    b = x.float()
    if wpost is not None:
        b = _rms(b) * wpost
    if scale is not None:
        b = b * scale
    new = r.float() + b
    return new.to(r.dtype), (_rms(new) * w).to(x.dtype)


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if own:
        from tsfast_amd import gated
    if kind == "step":
        step = gated.gated_recurrence_step if own else _plain_step
        return dict(o=step(s["q"], s["k"], s["v"], s["g"], s["state"]), state=s["state"])
    if kind in ("predict", "train"):
        recurrence = gated.gated_recurrence if own else _plain_recurrence
        o, last = recurrence(s["q"], s["k"], s["v"], s["g"], s["state"])
        out, given = dict(o=o, last=last), dict(o=s.get("do"), last=s.get("dstate"))
    elif kind == "gnorm":
        if own:
            y = gated.gated_norm(s["x"], s["gate"], s["w"], groups=c["groups"], eps=_EPS, gate_first=c["first"])
        else:
            y = _plain_gated_norm(s["x"], s["gate"], s["w"], c["groups"], c["first"])
        out, given = dict(y=y), dict(y=s.get("dy"))
    else:
        if own:
            new, y = gated.residual_norm(s["x"], s["r"], s["w"], post_weight=s["wpost"], scale=s["scale"], eps=_EPS)
        else:
            new, y = _plain_residual_norm(s["x"], s["r"], s["w"], s["wpost"], s["scale"])
        out, given = dict(r=new, y=y), dict(r=s.get("dr"), y=s.get("dy"))
    if "leaves" not in s:
        return out
    wanted = [n for n in out if given[n] is not None]
    grads = torch.autograd.grad([out[n] for n in wanted], s["leaves"], [given[n] for n in wanted])
    return dict({n: t.detach() for n, t in out.items()}, grads=list(grads))


# ------------------------------------------------------------------------------ bytes and flops


def work(case):
    c, kind = case, case["kind"]
    e = 2 if c["io"] == "bf16" else 4
    if kind == "step":
        B, H, Hk, K, V = (c[n] for n in ("B", "H", "Hk", "K", "V"))
        return dict(bytes=8 * B * H * K * V + e * B * (2 * Hk * K + 2 * H * V + H), flops=5 * B * H * K * V)
    if kind in ("predict", "train"):
        B, L, H, Hk, K, V = (c[n] for n in ("B", "L", "H", "Hk", "K", "V"))
        ins, state = e * B * L * (2 * Hk * K + H * V + H), 4 * B * H * K * V
        nbytes = ins + e * B * L * H * V + state * (2 if c["state"] else 1)
        flops = 4 * B * L * H * K * V
        if kind == "train":  # the incoming gradient read, the gradients written; the inputs once for both directions
            nbytes += e * B * L * H * V + ins + (2 * state if c["state"] else 0)
            flops += 10 * B * L * H * K * V
        return dict(bytes=nbytes, flops=flops)
    n, D = c["rows"] * c["D"], c["D"]
    if kind == "gnorm":
        return dict(bytes=e * n * (6 if c["train"] else 3) + 4 * D * (2 if c["train"] else 1), flops=n * (30 if c["train"] else 10))
    er = 2 if c["res"] == "bf16" else 4
    params = 4 * D * (1 + c["post"] + c["scale"])
    return dict(bytes=(2 * e + 2 * er) * n * (2 if c["train"] else 1) + params * (2 if c["train"] else 1),
                flops=n * (30 if c["train"] else 10))


# ------------------------------------------------------------------------------------- in 64 bits


def _exact_recurrence(s):
    """The recurrence step by step and, for a training pass, its adjoint, with the states of every
    64th step kept and those between computed again."""
    q, k, v, g = (s[n].detach().double() for n in ("q", "k", "v", "g"))
    B, L, H, V = v.shape
    Hk, K = q.shape[2:]
    R = H // Hk
    qh, kh = (t[:, :, :, None].expand(B, L, Hk, R, K).reshape(B, L, H, K) for t in (q, k))
    a = torch.exp(g)
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device=v.device) if s["state"] is None else s["state"].detach().double()
    every, kept, o = 64, [], torch.empty_like(v)

    def forward(S, t):
        S = a[:, t, :, None, None] * S
        return S.addcmul_(kh[:, t, :, :, None], v[:, t, :, None, :])

    train = "do" in s
    for t in range(L):
        if train and t % every == 0:
            kept.append(S)
        S = forward(S, t)
        o[:, t] = torch.matmul(qh[:, t, :, None], S)[:, :, 0]
    out = dict(o=o, last=S)
    if not train:
        return out
    do = s["do"].double()
    T = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double().clone()
    dq, dk, dv, dg = torch.empty_like(qh), torch.empty_like(kh), torch.empty_like(v), torch.empty_like(g)
    for c in range(len(kept) - 1, -1, -1):
        t0, t1 = c * every, min(L, (c + 1) * every)
        S, before, after = kept[c], [], []
        for t in range(t0, t1):
            before.append(S)
            S = forward(S, t)
            after.append(S)
        for t in range(t1 - 1, t0 - 1, -1):
            T = T.addcmul_(qh[:, t, :, :, None], do[:, t, :, None, :])
            dq[:, t] = torch.matmul(after[t - t0], do[:, t, :, :, None])[..., 0]
            dk[:, t] = torch.matmul(T, v[:, t, :, :, None])[..., 0]
            dv[:, t] = torch.matmul(kh[:, t, :, None], T)[:, :, 0]
            dg[:, t] = a[:, t] * (before[t - t0] * T).sum((-1, -2))
            T = a[:, t, :, None, None] * T
    dq, dk = (t.view(B, L, Hk, R, K).sum(3) for t in (dq, dk))
    return dict(out, grads=[dq, dk, dv, dg] + ([T] if s["state"] is not None else []))


def _exact_norm(x, weight, D):
    """The normalised rows, and what takes a gradient of them to the rows and the weight."""
    inv = (x.pow(2).sum(-1, keepdim=True) / D + _EPS).pow(-0.5)
    n = x * inv

    def back(dn):
        return inv * (dn - n * (dn * n).sum(-1, keepdim=True) / D)

    return n if weight is None else n * weight, n, back


def exact(case, seed):
    c, kind = case, case["kind"]
    s = prepare(case, seed)
    if kind in ("predict", "train"):
        return _exact_recurrence(s)
    if kind == "step":
        q, k, v, g, S = (s[n].double() for n in ("q", "k", "v", "g", "state"))
        R = v.shape[1] // q.shape[1]
        head = torch.arange(v.shape[1], device=v.device) // R
        S = torch.exp(g)[..., None, None] * S + torch.einsum("bhk,bhv->bhkv", k[:, head], v)
        return dict(o=torch.einsum("bhk,bhkv->bhv", q[:, head], S), state=S)
    D = c["D"]
    x, w = s["x"].detach().double(), s["w"].detach().double()
    if kind == "gnorm":
        G = c["groups"]
        shape = (-1, G, D // G)
        x, gate, w = x.view(shape), s["gate"].detach().double().view(shape), w.view(G, D // G)
        sig = 1 / (1 + torch.exp(-gate))
        act, dact = gate * sig, sig * (1 + gate * (1 - sig))
        y, n, back = _exact_norm(x * act if c["first"] else x, w, D // G)
        out = dict(y=(y if c["first"] else y * act).view(-1, D))
        if not c["train"]:
            return out
        dy = s["dy"].double().view(shape)
        if c["first"]:
            dp = back(dy * w)
            dx, dgate, dw = dp * act, dp * x * dact, (dy * n).sum(0)
        else:
            dx, dgate, dw = back(dy * w * act), dy * y * dact, (dy * n * act).sum(0)
        return dict(out, grads=[dx.reshape(-1, D), dgate.reshape(-1, D), dw.reshape(D)])
    r = s["r"].detach().double()
    wpost, scale = (None if s[n] is None else s[n].detach().double() for n in ("wpost", "scale"))
    if wpost is None:
        b = n1 = x
    else:
        b, n1, back1 = _exact_norm(x, wpost, D)
    new = r + (b if scale is None else b * scale)
    y, n, back = _exact_norm(new, w, D)
    out = dict(r=new, y=y)
    if not c["train"]:
        return out
    dy = s["dy"].double()
    dnew = s["dr"].double() + back(dy * w)
    db = dnew if scale is None else dnew * scale
    dx = db if wpost is None else back1(db * wpost)
    grads = [dx, dnew, (dy * n).sum(0)]
    if wpost is not None:
        grads.append((db * n1).sum(0))
    if scale is not None:
        grads.append((dnew * b).sum(0))
    return dict(out, grads=grads)
