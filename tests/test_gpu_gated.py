"""GPU parity of the gated linear recurrence and its step (HIP) against the float64 oracle.

Bars, relative to the largest value of each result, derived before the first run. float32: 1e-5, the package's bar (a float32
sum over 64 steps and up to 128 columns, and a state that decays, carry about 1e-6). bfloat16: an output is rounded
once, 2^-9 of its own size, and what is split into bfloat16 parts before it carries at most 2^-16: 2^-8 covers both.
The state stays float32: 2e-5 with bfloat16 inputs too (three parts of the decayed keys, 2^-24). g's gradient is a running sum
over at most 256 (float32) or 1024 (bfloat16) steps of terms that carry the products' errors, of either sign: it gets
3e-5, and 1e-2.
"""

import pytest
import torch

from oracle import gated_oracle as G
from tsfast_amd import _lib, dispatch, gated
from tsfast_amd.gated import core, recurrence_hip

pytestmark = pytest.mark.gpu

_DTYPES = [torch.float32, torch.bfloat16]


def _rel(a, b):
    if not b.numel():
        return 0.0
    assert torch.isfinite(a).all()
    return float((a.detach().cpu().double() - b).abs().max() / b.abs().max().clamp_min(1e-30))


def _inputs(B, L, H, Hk, K, V, dtype, seed=0, slow=0.05):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    g = -torch.rand(B, L, H, generator=r) * slow
    seq = (n(B, L, Hk, K), n(B, L, Hk, K) / K**0.5, n(B, L, H, V), g)
    return *(t.to("cuda", dtype) for t in seq), n(B, H, K, V).cuda(), n(B, L, H, V).to("cuda", dtype), n(B, H, K, V).cuda()


def _run(q, k, v, g, state, go, gl):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, state) if t is not None]
    with dispatch.use_backend("hip"):
        args = (*leaves[:4], leaves[4] if state is not None else None)
        assert dispatch.resolve("gated.recurrence", core._RECURRENCE_BACKENDS, (), args) is recurrence_hip
        o, last = gated.gated_recurrence(*args)
    outs, given = ([o, last], [go, gl]) if gl is not None else ([o], [go])
    return o, last, torch.autograd.grad(outs, leaves, given)


def _check(q, k, v, g, state, go, gl):
    o, last, grads = _run(q, k, v, g, state, go, gl)
    bf = v.dtype == torch.bfloat16
    tol, tol32, tolg = (2**-8, 2e-5, 1e-2) if bf else (1e-5, 1e-5, 3e-5)
    want_o, want_last, _ = G.recurrence(q, k, v, g, state)
    assert o.dtype == v.dtype and last.dtype == torch.float32
    assert _rel(o, want_o) < tol and _rel(last, want_last) < tol32
    wants = G.recurrence_grads(go, gl, q, k, v, g, state)
    for name, got, want, bar in zip("qkvgs", grads, wants, (tol, tol, tol, tolg, tol32)):
        assert got.shape == want.shape and _rel(got, want) < bar, name
    return o, last, grads


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize(
    "B,L,H,Hk,K,V",
    [
        (1, 1, 1, 1, 1, 1), (2, 2, 3, 1, 3, 5), (1, 16, 2, 2, 16, 16), (3, 63, 1, 1, 33, 17), (1, 64, 2, 2, 64, 64),
        (2, 65, 4, 2, 48, 80), (1, 128, 1, 1, 128, 128), (2, 129, 6, 3, 65, 127), (5, 200, 2, 1, 100, 24), (1, 300, 12, 4, 20, 128),
        (1, 1000, 1, 1, 128, 100), (1, 2050, 2, 1, 40, 72), (1, 511, 2, 2, 7, 128), (1, 512, 1, 1, 72, 8), (1, 513, 1, 1, 127, 65),
        (300, 70, 2, 2, 16, 16), (1, 1300, 2, 1, 33, 64), (2, 900, 1, 1, 64, 20), (1, 4000, 1, 1, 64, 100), (1, 700, 3, 3, 4, 6),
    ],
)
def test_matches_the_oracle(gpu, B, L, H, Hk, K, V, dtype):
    """Lengths about chunks, segments and anchors, widths about the tiles, shared heads, few rows and many."""
    _check(*_inputs(B, L, H, Hk, K, V, dtype, seed=L * 7 + K))


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("state,glast", [(False, False), (False, True), (True, False)])
def test_states_may_be_absent(gpu, state, glast, dtype):
    q, k, v, g, s, go, gl = _inputs(2, 150, 2, 2, 32, 48, dtype)
    _check(q, k, v, g, s if state else None, go, gl if glast else None)


def test_only_the_last_state_is_differentiated(gpu):
    q, k, v, g, s, go, gl = _inputs(1, 100, 2, 1, 16, 24, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, s)]
    grads = torch.autograd.grad(gated.gated_recurrence(*leaves)[1], leaves, gl)
    for got, want in zip(grads, G.recurrence_grads(torch.zeros_like(go), gl, q, k, v, g, s)):
        assert (want == 0).all() and (got == 0).all() or _rel(got, want) < 3e-5


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("L", [90, 700, 1500])
def test_gates_that_forget(gpu, L, dtype):
    """-inf, the type's lowest value and strong decays, at chunk borders too: no NaN, nothing leaks over them,
    and a gate that forgets has no gradient."""
    q, k, v, g, s, go, gl = _inputs(2, L, 3, 3, 32, 32, dtype)
    g[:, 0, 0] = float("-inf")
    g[:, 63::64, 0] = float("-inf")
    g[:, 64::192, 1] = torch.finfo(dtype).min
    g[0, 10:40, 2] = float("-inf")
    g[1, 20:80, 2] = -60.0
    _, _, grads = _check(q, k, v, g, s, go, gl)
    assert (grads[3][g < -104] == 0).all()
    v2 = v.clone()
    v2[0, :10] += 5  # before the run of -inf: nothing after it may change
    a, _ = gated.gated_recurrence(q, k, v, g, s)
    b, _ = gated.gated_recurrence(q, k, v2, g, s)
    assert torch.equal(a[0, 10:, 2], b[0, 10:, 2])


@pytest.mark.parametrize("dtype", _DTYPES)
def test_no_decay_and_padded_steps(gpu, dtype):
    """g = 0 adds everything up; steps with g = 0 and k = 0 pass the state on."""
    q, k, v, g, s, go, gl = _inputs(1, 257, 2, 2, 24, 40, dtype, slow=0.0)
    k[:, 100:170] = 0
    assert (g == 0).all()
    _check(q, k, v, g, s, go, gl)
    a = gated.gated_recurrence(q[:, :100], k[:, :100], v[:, :100], g[:, :100], s)[1]
    b = gated.gated_recurrence(q[:, :170], k[:, :170], v[:, :170], g[:, :170], s)[1]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", _DTYPES)
def test_zero_inputs_give_zeros(gpu, dtype):
    q, k, v, g, *_ = _inputs(1, 70, 1, 1, 16, 16, dtype)
    o, last = gated.gated_recurrence(torch.zeros_like(q), k, v, g)
    assert (o == 0).all() and torch.isfinite(last).all()
    o, last = gated.gated_recurrence(q, k, torch.zeros_like(v), g)
    assert (o == 0).all() and (last == 0).all()


@pytest.mark.parametrize("dtype", _DTYPES)
def test_empty_sequences_and_batches(gpu, dtype):
    q, k, v, g, s, go, gl = _inputs(2, 0, 2, 1, 8, 24, dtype)
    o, last, grads = _run(q, k, v, g, s, go, gl)
    assert o.shape == (2, 0, 2, 24) and torch.equal(last, s) and torch.equal(grads[4], gl)
    assert [t.shape for t in grads[:4]] == [q.shape, k.shape, v.shape, g.shape]
    assert (gated.gated_recurrence(q, k, v, g)[1] == 0).all()
    o, last = gated.gated_recurrence(*(t[:0] for t in _inputs(1, 5, 2, 1, 8, 24, dtype)[:4]))
    assert o.shape == (0, 5, 2, 24) and last.shape == (0, 2, 8, 24)


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("K,V", [(16, 24), (33, 15), (64, 128)])
def test_strides_and_alignment(gpu, K, V, dtype):
    """Slices of one projection at odd offsets, time-major tensors, expanded ones and a transposed last dimension give
    the contiguous tensors' bits."""
    B, L, H = 2, 140, 2
    q, k, v, g, s, go, gl = _inputs(B, L, H, H, K, V, dtype)
    both = torch.cat([torch.zeros(B, L, 1, device="cuda", dtype=dtype), *(t.flatten(2) for t in (q, k, v)), g], -1)
    n, views = 1, []
    for w, t in ((H * K, q), (H * K, k), (H * V, v), (H, g)):
        views.append(both[..., n : n + w].view(B, L, *t.shape[2:]))
        n += w
    time_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)]
    last = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v, g)]
    want = _run(q, k, v, g, s, go, gl)
    go_t, gl_t = go.transpose(0, 1).contiguous().transpose(0, 1), gl.mT.contiguous().mT
    for form in (views, time_major, last):
        o, last_s, grads = _run(*form, s.mT.contiguous().mT, go_t, gl_t)
        assert torch.equal(o, want[0]) and torch.equal(last_s, want[1])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[2]))
    wide = [t[:1].expand(B, *t.shape[1:]) for t in (q, k, v, g)]
    a, b = gated.gated_recurrence(*wide, s), gated.gated_recurrence(*(t.contiguous() for t in wide), s)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_broadcast_inputs_have_summed_gradients(gpu):
    q, k, v, g, *_, go, gl = _inputs(1, 80, 2, 2, 16, 16, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g)]
    o, last = gated.gated_recurrence(*(t.expand(3, *t.shape[1:]) for t in leaves))
    go3, gl3 = torch.randn(3, *go.shape[1:], device="cuda"), torch.randn(3, *gl.shape[1:], device="cuda")
    grads = torch.autograd.grad([o, last], leaves, [go3, gl3])
    wants = G.recurrence_grads(go3, gl3, *(t.expand(3, *t.shape[1:]) for t in (q, k, v, g)))
    for got, want in zip(grads, wants):
        assert _rel(got, want.sum(0, keepdim=True)) < 3e-5


def test_offsets_beyond_32_bits(gpu):
    """Rows that start more than 2^32 bytes into their buffer."""
    far = (1 << 31) + 4096
    big = torch.empty(far + 4096 * 40, device="cuda", dtype=torch.bfloat16)
    q, k, v, g, s, go, gl = _inputs(2, 70, 1, 1, 16, 16, torch.bfloat16)
    views, at = [], 0
    for t in (q, k, v, g):
        w = t.shape[-1] if t.dim() == 4 else 1
        view = big[at:].as_strided(t.shape, (far, 40, 40, 1)[: t.dim()])
        view.copy_(t)
        views.append(view)
        at += 4096 + 8 * w
    a, b = _run(*views, s, go, gl), _run(q, k, v, g, s, go, gl)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


def test_steps_far_apart_are_copied(gpu):
    """Steps beyond the 32-bit offsets of a chunk: the Python side copies, the library refuses."""
    q, k, v, g, s, go, gl = _inputs(1, 3, 1, 1, 16, 16, torch.bfloat16)
    far = recurrence_hip._MAX_STEP + 8
    big = torch.zeros(4 * far, device="cuda", dtype=torch.bfloat16)
    view = big.as_strided(v.shape, (3 * far, far, 16, 1))
    view.copy_(v)
    a, b = _run(q, k, view, g, s, go, gl), _run(q, k, v, g, s, go, gl)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))
    strides = recurrence_hip._Strides12(*q.stride()[:3], *k.stride()[:3], *view.stride()[:3], *g.stride())
    o, last = torch.empty_like(v), torch.empty_like(s)
    ptrs = [t.data_ptr() for t in (q, k, view, g)]
    status = _lib.load().tsfast_hip_gated_fwd(1, 3, 1, 1, 16, 16, 1, *ptrs, strides, None, o.data_ptr(), last.data_ptr(), None, 0, _lib.stream_of(v))
    assert status == -3


@pytest.mark.parametrize("dtype", _DTYPES)
def test_gradients_against_differences(gpu, dtype):
    """Central differences of the kernel's own forward over a random direction of each input, the loss summed in float64.
    A step of 1/8 along directions of the inputs' size: the loss is a polynomial of q, k, v and the state (exact for one
    input at a time up to second order), and exp's third order adds below 1e-2 for g's; bfloat16 outputs, rounded at 2^-9,
    leave noise of sqrt(outputs) 2^-9 on sums of as many terms."""
    q, k, v, g, s, go, gl = _inputs(2, 150, 2, 1, 24, 32, dtype)
    g = g - 0.1  # no decay near 0, where a step would cross it
    _, _, grads = _run(q, k, v, g, s, go, gl)

    def loss(*a):
        o, last = gated.gated_recurrence(*a)
        return float((o.double() * go.double()).sum() + (last.double() * gl.double()).sum())

    r = torch.Generator().manual_seed(11)
    for n, t in enumerate((q, k, v, g, s)):
        d = torch.randn(t.shape, generator=r).to(t) * (0.5 if n < 3 else 0.02 if n == 3 else 0.5)
        ends = []
        for sign in (1, -1):
            moved = [q, k, v, g, s]
            moved[n] = (t.double() + sign * 0.125 * d.double()).to(t.dtype)
            ends.append((moved[n].double(), loss(*moved)))
        step = ends[0][0] - ends[1][0]  # what rounding made of it
        want, got = ends[0][1] - ends[1][1], float((grads[n].double() * step).sum())
        scale = float((grads[n].double() * step).norm())  # of a sum of such terms with random signs
        noise = 0.0 if dtype == torch.float32 else 2**-8 * float(go.double().norm()) * float(v.double().abs().mean()) * 2
        assert abs(got - want) < 0.05 * scale + 0.01 * abs(want) + noise, n


@pytest.mark.parametrize("dtype", _DTYPES)
def test_repeats_give_the_same_bits(gpu, dtype):
    """The same call twice gives the same bits: no atomics."""
    args = _inputs(2, 600, 4, 2, 32, 48, dtype)
    a, b = _run(*args), _run(*args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@pytest.mark.parametrize("dtype", _DTYPES)
def test_pieces_of_a_row_carry_the_state(gpu, dtype):
    """Truncated passes with the state carried equal the whole pass, and so do single steps."""
    q, k, v, g, s, *_ = _inputs(2, 150, 4, 2, 32, 24, dtype)
    o, last = gated.gated_recurrence(q, k, v, g, s)
    S, outs = s, []
    for lo, hi in ((0, 1), (1, 65), (65, 129), (129, 150)):
        y, S = gated.gated_recurrence(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], g[:, lo:hi], S)
        outs.append(y)
    tol = 2**-7 if dtype == torch.bfloat16 else 2e-5  # two results, each within its own bar
    assert _rel(torch.cat(outs, 1), o.cpu().double()) < tol and _rel(S, last.cpu().double()) < 4e-5
    S, outs = s.clone(), []
    for t in range(150):
        outs.append(gated.gated_recurrence_step(q[:, t], k[:, t], v[:, t], g[:, t], S))
    assert _rel(torch.stack(outs, 1), o.cpu().double()) < tol and _rel(S, last.cpu().double()) < 4e-5


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("L,H,Hk,K,V", [(1500, 4, 2, 24, 100), (700, 2, 2, 100, 24), (70, 2, 1, 16, 16)])
def test_states_kept_for_the_backward(gpu, L, H, Hk, K, V, dtype):
    """The backward with the forward's states between segments (none where rows are whole) and without, and again."""
    q, k, v, g, state, go, gl = _inputs(2, L, H, Hk, K, V, dtype)
    leaves = [t.requires_grad_() for t in (q, k, v, g, state)]
    o, last = recurrence_hip.run(*leaves)
    first = torch.autograd.grad([o, last], leaves, [go, gl], retain_graph=True)
    again = torch.autograd.grad([o, last], leaves, [go, gl])
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with torch.no_grad():
        _, _, kept = recurrence_hip._recurrence_train_op(q, k, v, g, state)
        assert (kept.numel() > 0) == (L > 256)
        without = recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, state)
        assert all(torch.equal(a, b) for a, b in zip(first, recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, state, kept)))
        with pytest.raises(TypeError, match="kept"):
            recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, state, kept.new_empty(kept.numel() + 16))
    bf = dtype == torch.bfloat16
    bars = (2**-8, 2**-8, 2**-8, 1e-2, 2e-5) if bf else (1e-5, 1e-5, 1e-5, 3e-5, 1e-5)
    for got, want, bar in zip(without, G.recurrence_grads(go, gl, q, k, v, g, state), bars):
        assert _rel(got, want) < bar


@pytest.mark.parametrize("dtype", _DTYPES)
@pytest.mark.parametrize("B,H,Hk,K,V", [(1, 1, 1, 1, 1), (1, 4, 2, 64, 64), (3, 6, 2, 33, 17), (2, 5, 5, 200, 130), (600, 2, 1, 128, 128),
                                        (300, 2, 2, 7, 65), (1, 2, 1, 1024, 3)])
def test_step_matches_the_oracle(gpu, B, H, Hk, K, V, dtype):
    q, k, v, g, s, *_ = _inputs(B, 1, H, Hk, K, V, dtype, slow=2.0)
    g[0, 0, 0] = float("-inf")
    want_o, want_s, _ = G.recurrence(q, k, v, g, s)
    where = s.data_ptr()
    with dispatch.use_backend("hip"):
        o = gated.gated_recurrence_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s)
    tol = 2**-8 if dtype == torch.bfloat16 else 1e-5
    assert s.data_ptr() == where and o.dtype == dtype and _rel(o, want_o[:, 0]) < tol and _rel(s, want_s) < 1e-6


def test_step_strides_versions_and_refusals(gpu):
    q, k, v, g, s, *_ = _inputs(3, 4, 2, 1, 16, 24, torch.float32)
    want = s.clone()
    a = gated.gated_recurrence_step(*(t[:, 2].contiguous() for t in (q, k, v, g)), want)
    version = s._version
    b = gated.gated_recurrence_step(q[:, 2], k[:, 2], v[:, 2], g[:, 2], s)
    assert torch.equal(a, b) and torch.equal(s, want) and s._version > version
    last = [t[:, 2].transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]
    assert recurrence_hip.supports_step(*last, g[:, 2], s) is None
    assert "contiguous" in recurrence_hip.supports_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s.mT.contiguous().mT)
    assert "float32 state" in recurrence_hip.supports_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s.double())
    with pytest.raises(RuntimeError, match="no gradient"):
        gated.gated_recurrence_step(q[:, 2].requires_grad_(), k[:, 2], v[:, 2], g[:, 2], s)
    with torch.inference_mode():
        gated.gated_recurrence_step(q[:, 2], k[:, 2], v[:, 2], g[:, 2], s.clone())


def test_supports_reasons(gpu):
    q, k, v, g, s, *_ = _inputs(1, 5, 2, 1, 8, 8, torch.float32)
    ok = recurrence_hip.supports
    assert ok(q, k, v, g, s) is None and ok(q, k, v, g, None) is None
    assert "GPU-only" in ok(q.cpu(), k.cpu(), v.cpu(), g.cpu(), None)
    assert "q dtype" in ok(q.bfloat16(), k, v, g, None)
    assert "float32 state" in ok(q, k, v, g, s.bfloat16())
    assert "outside" in ok(q, k, torch.zeros(1, 5, 2, 129, device="cuda"), g, None)
    wide = torch.randn(1, 5, 2, 130, device="cuda")
    o, _ = gated.gated_recurrence(q, k, wide, g)  # served by the torch path
    assert _rel(o, G.recurrence(q, k, wide, g)[0]) < 1e-5


@pytest.mark.parametrize("dtype", _DTYPES)
def test_other_streams_and_graphs(gpu, dtype):
    """On a side stream, and captured: replays on new inputs, with eager work between them, equal the eager result."""
    args = _inputs(2, 520, 2, 1, 32, 40, dtype)
    want = _run(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(*args)
        got = _run(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
    q, k, v, g, s, go, gl = (t.clone() for t in args)
    step_state = s.clone()

    def work():
        o, last = recurrence_hip._recurrence_op(q, k, v, g, s)
        grads = recurrence_hip._recurrence_bwd_op(go, gl, q, k, v, g, s)
        y = gated.gated_recurrence_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], step_state)
        return o, last, *grads, y

    with torch.no_grad():
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work()
        for seed in (1, 2, 3):
            for dst, src in zip((q, k, v, g, s, go, gl), _inputs(2, 520, 2, 1, 32, 40, dtype, seed=seed)):
                dst.copy_(src)
            step_state.copy_(s)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs] + [step_state.clone()]
            step_state.copy_(s)
            eager = [*work(), step_state]
            assert all(torch.equal(a, b) for a, b in zip(got, eager)), seed


def test_compile_traces_the_recurrence(gpu):
    q, k, v, g, s, go, gl = _inputs(1, 70, 2, 1, 16, 16, torch.float32)

    def f(q, k, v, g, s):
        o, last = gated.gated_recurrence(q * 1.5, k, v, g, s)
        return (o * 2).sum() + last.sum()

    grads = []
    for fn in (f, torch.compile(f, fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, g, s)]
        grads.append(torch.autograd.grad(fn(*leaves), leaves))
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
