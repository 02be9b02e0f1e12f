"""The operators of a selective state space layer in service and of the feed-forward block behind it,
each as one pass that a program of this package makes.

``gated_feed_forward`` is the block's two projections, the activation and their product, in training and for
prompts and tokens; ``mamba_conv_packed`` and ``mamba_ssm_packed`` are the layer's short causal convolution and
its scan over prompts of different lengths packed into one row, with the states they leave; ``mamba_step`` is
everything between the layer's input and output projections for one token of each sequence, with the states in
place. With ``own`` the calls are the package's; without, the same operators in elementary torch operations in
float32. ``exact`` is the definition in float64.

Widths and lengths are those of the package's benchmark (batch 16, length 4096, width 1536, 16 states) and of
identification models (windows of 512, widths of 64 to 256), with the odd sizes such models come to.
"""

from __future__ import annotations

import math

import torch

own = False

_IO = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the feed-forward block behind one token of one sequence: a read of both weights
        dict(name="feed_token", kind="feed", rows=1, D=1536, F=4096, io="bf16", act="silu", bias=False, train=False),
        # the same for one token of each of a batch of served sequences
        dict(name="feed_serving", kind="feed", rows=256, D=1536, F=4096, io="bf16", act="silu", bias=False, train=False),
        # a prompt through a narrow model of odd widths
        dict(name="feed_odd", kind="feed", rows=777, D=195, F=517, io="fp32", act="gelu", bias=True, train=False),
        # a training step on a batch of windows, an identification model's width
        dict(name="feed_windows", kind="feed", rows=32768, D=64, F=256, io="fp32", act="sigmoid", bias=True, train=True),
        # a training step at the benchmark's batch, length and width
        dict(name="feed_large", kind="feed", rows=65536, D=1536, F=4096, io="bf16", act="silu", bias=False, train=True),
        # one sample of one model running on-line
        dict(name="step_online", kind="step", B=1, D=128, N=16, R=8, K=4, io="fp32"),
        # one token for each of a batch of served sequences, at the benchmark's width
        dict(name="step_serving", kind="step", B=256, D=1536, N=16, R=96, K=4, io="bf16"),
        # the first window of a session: one short prompt before the steps
        dict(name="conv_prompt", kind="conv", T=77, S=1, D=128, K=4, io="fp32", carried=False, empty=False, behind=0),
        # prompts of a batch of sessions that go on (their tails carried in), some of no or one token, in a buffer with room behind
        dict(name="conv_prompts", kind="conv", T=16384, S=24, D=1536, K=4, io="bf16", carried=True, empty=True, behind=100),
        # the scans of the same two
        dict(name="scan_prompt", kind="scan", T=77, S=1, D=128, N=16, io="fp32", carried=False, empty=False, behind=0),
        dict(name="scan_prompts", kind="scan", T=16384, S=24, D=1536, N=16, io="bf16", carried=True, empty=True, behind=100),
        # a whole recording through a narrow model before it is predicted on-line: one sequence and a long time axis
        dict(name="scan_recording", kind="scan", T=65536, S=1, D=256, N=16, io="bf16", carried=False, empty=False, behind=0),
    ]


# ---------------------------------------------------------------------------------- drawn sizes


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A width of [lo, hi], most often a multiple of 32 or 8."""
    step = rng.choice([32, 32, 8, 1])
    return max(lo, _log(rng, lo, hi) // step * step)


def _draw_once(rng):
    kind = rng.choice(["feed", "feed", "feed", "step", "step", "conv", "scan", "scan"])
    io = rng.choice(["fp32", "bf16"])
    if kind == "feed":
        train = rng.random() < 0.5
        D = _width(rng, 32, 2048)
        step = rng.choice([64, 8, 1])
        F = min(8192, max(32, int(D * rng.choice([1, 2, 8 / 3, 4])) // step * step))
        rows = _log(rng, 100, 65536) if train else _log(rng, 1, 16384)
        return dict(kind=kind, rows=rows, D=D, F=F, io=io, act=rng.choice(["silu", "gelu", "sigmoid"]), bias=rng.random() < 0.5, train=train)
    if kind == "step":
        D = _width(rng, 32, 2048)
        return dict(kind=kind, B=_log(rng, 1, 256), D=D, N=rng.choice([8, 16, 16, 16, 32, 64, rng.randint(3, 40)]), R=max(1, -(-D // 16)),
                    K=rng.choice([4, 4, 4, 2, 3]), io=io)
    T, S = _log(rng, 20, 65536), _log(rng, 1, 64)
    S = min(S, T // 4)
    common = dict(kind=kind, T=T, S=S, D=_width(rng, 32, 2048), io=io, carried=rng.random() < 0.5, empty=S > 4 and rng.random() < 0.5,
                  behind=rng.choice([0, 0, T // 10]))
    if kind == "conv":
        return dict(common, K=rng.choice([4, 4, 4, 2, 3]))
    return dict(common, N=rng.choice([8, 16, 16, 16, 32, 64, rng.randint(3, 40)]))


def _size(case):
    """A rough cost of one pass against the largest listed of its kind."""
    c = case
    if c["kind"] == "feed":
        products = c["rows"] * c["D"] * c["F"] * (3 if c["train"] else 1) / (65536 * 1536 * 4096 * 3)
        return max(products * (8 if c["io"] == "fp32" else 1), c["rows"] * c["F"] / (65536 * 4096))
    if c["kind"] == "step":
        return c["B"] * c["D"] * c["N"] / (256 * 2048 * 64)
    return c["T"] * c["D"] * c.get("N", 16) / (16384 * 1536 * 16)


def draw(rng):
    while True:
        case = _draw_once(rng)
        if _size(case) <= 1.0:
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


def _starts(r, c):
    """Where the sequences begin and end in a row of T tokens: random lengths; with ``empty``, among them one of no token and one of one."""
    used, S = c["T"] - c["behind"], c["S"]
    cuts = r.uniform(0, used, S - 1).long().sort().values if S > 1 else torch.empty(0, dtype=torch.long, device="cuda")
    starts = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), used)])
    if c["empty"]:
        starts[2] = starts[1]
        starts[4] = torch.minimum(starts[3] + 1, starts[5])
    return starts.to(torch.int32)


def _step_sizes(r, *shape):
    """What goes into the softplus: step sizes of a trained layer, 1e-3 to 0.1 with a spread per token."""
    D = shape[-1]
    base = torch.exp(r.uniform(math.log(1e-3), math.log(0.1), D))
    return torch.log(torch.expm1(base)) + 0.5 * r.normal(*shape)


def _rates(r, D, N):
    """The states' rates: -1 .. -N with a spread per channel."""
    return -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * r.uniform(0.5, 1.5, D, 1)


def prepare(case, seed):
    r, c, kind = _Inputs(seed), case, case["kind"]
    dt = _IO[c["io"]]
    s = dict(case=dict(c))
    if kind == "feed":
        rows, D, F = c["rows"], c["D"], c["F"]
        s.update(x=r.normal(rows, D, dtype=dt), wg=(r.normal(F, D) / math.sqrt(D)).to(dt), wu=(r.normal(F, D) / math.sqrt(D)).to(dt))
        s.update(bg=(0.3 * r.normal(F)).to(dt) if c["bias"] else None, bu=(0.3 * r.normal(F)).to(dt) if c["bias"] else None)
        if c["train"]:
            s["dy"] = r.normal(rows, F, dtype=dt)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "wg", "wu", "bg", "bu") if s[n] is not None]
    elif kind == "step":
        B, D, N, R, K = (c[n] for n in ("B", "D", "N", "R", "K"))
        s.update(x=r.normal(B, D, dtype=dt), z=r.normal(B, D, dtype=dt), tail=r.normal(B, D, K - 1, dtype=dt), h=r.normal(B, D, N))
        s.update(wc=(r.normal(D, 1, K) / math.sqrt(K)).to(dt), bc=(0.1 * r.normal(D)).to(dt))
        s.update(xp=(2 * r.normal(R + 2 * N, D) / math.sqrt(D)).to(dt), dp=(r.normal(D, R) * R**-0.5).to(dt), db=_step_sizes(r, D))
        s.update(A=_rates(r, D, N), Dp=1 + 0.2 * r.normal(D))
    else:
        T, S, D = c["T"], c["S"], c["D"]
        s["starts"] = _starts(r, c)
        if kind == "conv":
            K = c["K"]
            s.update(x=r.normal(T, D, dtype=dt), wc=(r.normal(D, 1, K) / math.sqrt(K)).to(dt), bc=(0.1 * r.normal(D)).to(dt))
            s["tails"] = r.normal(S, D, K - 1, dtype=dt) if c["carried"] else None
        else:
            N = c["N"]
            s.update(draw=_step_sizes(r, T, D).to(dt), A=_rates(r, D, N), Bt=r.normal(T, N, dtype=dt), Ct=r.normal(T, N, dtype=dt),
                     u=r.normal(T, D, dtype=dt), z=r.normal(T, D, dtype=dt), Dp=1 + 0.2 * r.normal(D))
            s["h0"] = r.normal(S, D, N) if c["carried"] else None
    return s


# ----------------------------------------------------------------------------------- the passes


def _silu(x):
    return x * torch.sigmoid(x)


def _activation(a, act):
    if act == "silu":
        return _silu(a)
    if act == "sigmoid":
        return torch.sigmoid(a)
    return 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _plain_feed(x, wg, wu, bg, bu, act):
    a, b = x.float() @ wg.float().T, x.float() @ wu.float().T
    if bg is not None:
        a, b = a + bg.float(), b + bu.float()
    return (_activation(a, act) * b).to(x.dtype)


def _plain_step(x, z, tail, h, wc, bc, xp, dp, db, A, Dp):
    N, R = h.shape[-1], dp.shape[-1]
    window = torch.cat([tail, x[..., None]], -1)
    u = _silu((window.float() * wc[:, 0].float()).sum(-1) + bc.float())
    dt, Bt, Ct = (u @ xp.float().T).split([R, N, N], -1)
    delta = _softplus(dt @ dp.float().T + db)
    new = torch.exp(delta[..., None] * A) * h + (delta * u)[..., None] * Bt[:, None]
    y = ((new * Ct[:, None]).sum(-1) + Dp * u) * _silu(z.float())
    h.copy_(new)
    tail.copy_(window[..., 1:])
    return y.to(x.dtype)


def _which(starts, T):
    """Each token's sequence, and whether it has one."""
    at = torch.arange(T, device=starts.device)
    return torch.searchsorted(starts.long(), at, right=True) - 1, at < starts[-1]


def _plain_conv(x, starts, wc, bc, tails):
    T, D = x.shape
    S, K = starts.shape[0] - 1, wc.shape[-1]
    if tails is None:
        tails = x.new_zeros(S, D, K - 1)
    seq, live = _which(starts, T)
    # every sequence behind its K - 1 carried tokens
    room = torch.zeros(T + (S + 1) * (K - 1), D, device=x.device)
    place = torch.arange(T, device=x.device) + (seq + 1) * (K - 1)
    room[place] = x.float()
    back = torch.arange(K - 1, device=x.device)
    first = starts[:-1].long() + torch.arange(S, device=x.device) * (K - 1)
    room[first[:, None] + back] = tails.float().transpose(1, 2)
    taps = torch.stack([room[place - (K - 1) + k] * wc[:, 0, k].float() for k in range(K)])
    u = torch.where(live[:, None], _silu(taps.sum(0) + bc.float()), 0.0)
    last = starts[1:].long() + torch.arange(S, device=x.device) * (K - 1)
    return u.to(x.dtype), room[last[:, None] + back].transpose(1, 2).to(x.dtype).contiguous()


def _plain_scan(draw, A, Bt, Ct, u, z, Dp, starts, h0):
    T, D = draw.shape
    S, N = starts.shape[0] - 1, A.shape[-1]
    seq, live = _which(starts, T)
    delta = torch.where(live[:, None], _softplus(draw.float()), 0.0)
    decay = torch.exp(delta[..., None] * A)
    h = (delta * u.float())[..., None] * Bt.float()[:, None]
    # a sequence begins with its own state and keeps nothing of the one before it
    begins = live & (torch.arange(T, device=draw.device) == starts.long()[seq])
    if h0 is not None:
        h = h + torch.where(begins[:, None, None], decay * h0[seq.clamp(max=S - 1)], 0.0)
    decay = torch.where(begins[:, None, None], 0.0, decay)
    span = 1
    while span < T:
        h = torch.cat([h[:span], h[span:] + decay[span:] * h[:-span]])
        decay = torch.cat([decay[:span], decay[span:] * decay[:-span]])
        span *= 2
    y = ((h * Ct.float()[:, None]).sum(-1) + Dp * u.float()) * _silu(z.float())
    ends, some = starts[1:].long() - 1, starts[1:] > starts[:-1]
    before = torch.zeros(S, D, N, device=draw.device) if h0 is None else h0
    last = torch.where(some[:, None, None], h[ends.clamp(min=0)], before)
    return torch.where(live[:, None], y, 0.0).to(draw.dtype), last


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if own:
        from tsfast_amd import gated, mamba
    if kind == "feed":
        if own:
            y = gated.gated_feed_forward(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["act"])
        else:
            y = _plain_feed(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], c["act"])
        if "leaves" not in s:
            return dict(y=y)
        return dict(y=y.detach(), grads=list(torch.autograd.grad(y, s["leaves"], s["dy"])))
    if kind == "step":
        step = mamba.mamba_step if own else _plain_step
        y = step(s["x"], s["z"], s["tail"], s["h"], s["wc"], s["bc"], s["xp"], s["dp"], s["db"], s["A"], s["Dp"])
        return dict(y=y, tail=s["tail"], h=s["h"])
    if kind == "conv":
        conv = mamba.mamba_conv_packed if own else _plain_conv
        u, tails = conv(s["x"], s["starts"], s["wc"], s["bc"], s["tails"])
        return dict(u=u, tails=tails)
    scan = mamba.mamba_ssm_packed if own else _plain_scan
    y, last = scan(s["draw"], s["A"], s["Bt"], s["Ct"], s["u"], s["z"], s["Dp"], s["starts"], s["h0"])
    return dict(y=y, last=last)


# ------------------------------------------------------------------------------ bytes and flops


def work(case):
    c, kind = case, case["kind"]
    e = 2 if c["io"] == "bf16" else 4
    if kind == "feed":
        rows, D, F = c["rows"], c["D"], c["F"]
        weights = e * (2 * F * D + (2 * F if c["bias"] else 0))
        nbytes, flops = e * rows * (D + F) + weights, 4 * rows * D * F
        if c["train"]:  # the incoming gradient read, the inputs' gradients written; the inputs once for both directions
            nbytes += e * rows * (D + F) + weights
            flops *= 3
        return dict(bytes=nbytes, flops=flops)
    if kind == "step":
        B, D, N, R, K = (c[n] for n in ("B", "D", "N", "R", "K"))
        weights = e * (D * K + D + (R + 2 * N) * D + D * R) + 4 * (2 * D + D * N)
        return dict(bytes=weights + B * D * (8 * N + e * (2 * (K - 1) + 3)), flops=B * D * (2 * K + 2 * (2 * R + 2 * N) + 7 * N))
    T, S, D = c["T"] - c["behind"], c["S"], c["D"]
    if kind == "conv":
        K = c["K"]
        states = e * S * D * (K - 1) * (2 if c["carried"] else 1)
        return dict(bytes=e * (T * D + c["T"] * D + D * K + D) + states, flops=T * D * (2 * K + 4))
    N = c["N"]
    states = 4 * S * D * N * (2 if c["carried"] else 1)
    return dict(bytes=e * (T * (3 * D + 2 * N) + c["T"] * D) + 4 * (D * N + D) + states, flops=T * D * (7 * N + 12))


# ------------------------------------------------------------------------------------- in 64 bits


def _exact_feed(s, act):
    x, wg, wu = (s[n].detach().double() for n in ("x", "wg", "wu"))
    a, b = torch.nn.functional.linear(x, wg), torch.nn.functional.linear(x, wu)
    if s["bg"] is not None:
        a += s["bg"].detach().double()
        b += s["bu"].detach().double()
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-a / math.sqrt(2.0))
        f, df = a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    else:
        sig = 1 / (1 + torch.exp(-a))
        f, df = (a * sig, sig + a * sig * (1 - sig)) if act == "silu" else (sig, sig * (1 - sig))
    y = f * b
    if "dy" not in s:
        return dict(y=y)
    dy = s["dy"].double()
    da, db = dy * b * df, dy * f
    grads = [torch.mm(da, wg) + torch.mm(db, wu), torch.mm(da.T, x), torch.mm(db.T, x)]
    if s["bg"] is not None:
        grads += [da.sum(0), db.sum(0)]
    return dict(y=y, grads=grads)


def _exact_step(s):
    x, z, tail, h, wc, bc, xp, dp, db, A, Dp = (s[n].double() for n in ("x", "z", "tail", "h", "wc", "bc", "xp", "dp", "db", "A", "Dp"))
    K, N, R = wc.shape[-1], h.shape[-1], dp.shape[-1]
    pre = bc + wc[:, 0, K - 1] * x
    for k in range(K - 1):
        pre = pre + wc[:, 0, k] * tail[..., k]
    u = pre / (1 + torch.exp(-pre))
    p = torch.mm(u, xp.T)
    delta = torch.nn.functional.softplus(torch.mm(p[:, :R], dp.T) + db)
    h = h * torch.exp(torch.einsum("bd,dn->bdn", delta, A)) + torch.einsum("bd,bn->bdn", delta * u, p[:, R : R + N])
    y = (torch.einsum("bdn,bn->bd", h, p[:, R + N :]) + Dp * u) * z / (1 + torch.exp(-z))
    return dict(y=y, tail=torch.cat((tail[..., 1:], x[..., None]), -1), h=h)


def _bounds(s):
    at = s["starts"].tolist()
    return list(zip(at[:-1], at[1:]))


def _exact_conv(s):
    x, wc, bc = s["x"].double(), s["wc"].double(), s["bc"].double()
    K, D = wc.shape[-1], x.shape[-1]
    u, tails = torch.zeros_like(x), []
    for n, (t0, t1) in enumerate(_bounds(s)):
        before = x.new_zeros(D, K - 1) if s["tails"] is None else s["tails"][n].double()
        row = torch.cat([before, x[t0:t1].T], 1)
        tails.append(row[:, row.shape[1] - (K - 1) :])
        if t1 > t0:
            pre = (bc[:, None] + sum(wc[:, 0, k, None] * row[:, k : k + t1 - t0] for k in range(K))).T
            u[t0:t1] = pre / (1 + torch.exp(-pre))
    return dict(u=u, tails=torch.stack(tails))


def _exact_scan(s):
    """Step by step, all sequences side by side as long as each lasts."""
    draw, A, Bt, Ct, u, z, Dp = (s[n].double() for n in ("draw", "A", "Bt", "Ct", "u", "z", "Dp"))
    bounds = _bounds(s)
    h = draw.new_zeros(len(bounds), *A.shape) if s["h0"] is None else s["h0"].double().clone()
    delta = torch.nn.functional.softplus(draw)
    y = torch.zeros_like(draw)
    order = sorted(range(len(bounds)), key=lambda n: bounds[n][0] - bounds[n][1])  # the longest first
    rank = torch.tensor(order, device=draw.device)
    begin = s["starts"].long()[:-1][rank]
    lengths = sorted((t1 - t0 for t0, t1 in bounds), reverse=True)
    state = h[rank]
    n = len(order)
    for i in range(lengths[0]):
        while lengths[n - 1] <= i:
            n -= 1
        t = begin[:n] + i
        d = delta[t]
        state[:n] = torch.addcmul((d * u[t])[..., None] * Bt[t][:, None], torch.exp(d[..., None] * A), state[:n])
        y[t] = torch.matmul(state[:n], Ct[t][..., None])[..., 0]
    h[rank] = state
    y = (y + Dp * u) * z / (1 + torch.exp(-z))
    y[bounds[-1][1] :] = 0
    return dict(y=y, last=h)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "feed":
        return _exact_feed(s, case["act"])
    return {"step": _exact_step, "conv": _exact_conv, "scan": _exact_scan}[kind](s)
