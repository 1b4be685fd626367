"""apply_rotary_positions on the GPU against the float64 oracle.

Tolerance: one rounding to the 16-bit type (half a step, eps / 2 of the
result) and the fp32 arithmetic before it: cosine and sine within 3e-7 (fp32
polynomials of an angle rounded to 24 bits, at most pi/4) and two products and
a sum, 3 roundings of 2^-24, so 5e-7 of m (|a| + |b|).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as orc

pytestmark = pytest.mark.gpu

YARN = {"type": "yarn", "factor": 8, "original_length": 8192}
WAVE = {"type": "wavelength", "factor": 8, "original_length": 8192, "low": 1, "high": 4}

CASES = [
    # (B, S, H, Hk, D, R, interleaved, scaling, dtype, first position)
    (1, 1, 1, 1, 64, 64, False, None, torch.float16, 0),
    (2, 37, 8, 2, 128, 128, False, YARN, torch.bfloat16, 5),
    (3, 5, 4, 4, 64, 16, True, WAVE, torch.float16, 70001),
    (1, 1100, 3, 1, 32, 24, False, {"type": "ntk", "factor": 4}, torch.bfloat16, 0),
    (2, 9, 2, 2, 16, 8, False, {"type": "linear", "factor": 3}, torch.float16, 1000003),
    (1, 7, 5, 1, 128, 10, False, None, torch.float16, 2 ** 30),       # unaligned pairs
    (1, 7, 5, 1, 64, 6, True, None, torch.bfloat16, -12),             # part of a chunk, negative
    (1, 3, 2, 1, 256, 256, True, None, torch.float16, 9),
    (1, 4, 3, 2, 8, 2, False, None, torch.float16, 3),
    (5, 1, 32, 8, 128, 96, False, {"type": "factors", "factors": [1.0 + 0.1 * i for i in range(48)],
                                   "attention_factor": 1.2}, torch.bfloat16, 131071),
    (1, 2051, 2, 1, 64, 64, False, None, torch.float16, 100),         # 4 tokens a workgroup, ragged
]


def _inputs(B, S, heads, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((B, S, heads, D), generator=g).to(dtype)


def _check(got, x, pos, rot, inverse, what):
    """got against the oracle's rotation of x (CPU tensors)."""
    ref = orc.rotate(x.double().numpy(), pos, rot.frequencies, rot.attention_factor,
                     rot.interleaved, inverse)
    mag = orc.rotate(np.abs(x.double().numpy()), pos * 0, rot.frequencies, rot.attention_factor,
                     rot.interleaved)                        # m |own|
    R = rot.rotary_dim
    other = mag.copy()
    a, b = ((slice(0, R, 2), slice(1, R, 2)) if rot.interleaved
            else (slice(0, R // 2), slice(R // 2, R)))
    other[..., a], other[..., b] = mag[..., b], mag[..., a]
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    tol = torch.finfo(x.dtype).eps / 2 * np.abs(ref) * 1.0001 + 5e-7 * (mag + other) + tiny
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"{what}: {(err / tol).max():.3g} times the tolerance"
    assert torch.equal(got.cpu()[..., R:], x[..., R:]), f"{what}: columns from {R} on changed"


@pytest.mark.parametrize("B,S,H,Hk,D,R,inter,scaling,dtype,first", CASES)
@pytest.mark.parametrize("layout,wide", [("bshd", False), ("bhsd", True)])
def test_forward_and_backward(B, S, H, Hk, D, R, inter, scaling, dtype, first, layout, wide):
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    print(f"[case] rotary {B} {S} {H} {Hk} {D} R={R} {inter} {dtype} {layout}", flush=True)
    rot = RotaryPositions(R, base=10000.0, interleaved=inter, scaling=scaling)
    cpu = [_inputs(B, S, h, D, dtype, 3 + i) for i, h in enumerate((H, Hk, H, Hk))]
    if layout == "bhsd":
        q, k, gq, gk = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in cpu)
    else:
        q, k, gq, gk = (t.cuda() for t in cpu)
    pos = first + np.arange(S)[None] + 3 * np.arange(B)[:, None]
    positions = torch.tensor(pos, dtype=torch.int64 if wide else torch.int32, device="cuda")
    q.requires_grad_()
    k.requires_grad_()
    qo, ko = apply_rotary_positions(q, k, positions, rot)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    for got, x, inverse, what in ((qo, cpu[0], False, "q"), (ko, cpu[1], False, "k"),
                                  (dq, cpu[2], True, "dq"), (dk, cpu[3], True, "dk")):
        assert got.is_contiguous() and got.dtype == dtype
        _check(got.detach(), x, pos, rot, inverse, what)


@pytest.mark.parametrize("D,R,inter", [(24, 16, True), (24, 24, False), (40, 32, False), (40, 8, False),
                                       (48, 48, False), (96, 64, True), (80, 18, False)])
def test_other_head_dims(D, R, inter):
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    rot = RotaryPositions(R, interleaved=inter)
    x = _inputs(2, 11, 3, D, torch.float16, D)
    pos = 40 + np.arange(11)[None] + np.zeros((2, 1), dtype=np.int64)
    got = apply_rotary_positions(x.cuda(), None, torch.arange(40, 51, device="cuda"), rot)[0]
    _check(got, x, pos, rot, False, "x")


def test_gradients_of_expanded_and_wide_upstreams():
    """A sum's gradient (strides of 0) and an fp32 one are taken."""
    from flash_attn_volta import RotaryPositions, apply_rotary_positions, rotary_backward
    rot = RotaryPositions(64)
    pos = torch.arange(5, device="cuda")
    x = _inputs(1, 5, 2, 64, torch.float16, 0).cuda().requires_grad_()
    apply_rotary_positions(x, None, pos, rot)[0].sum().backward()
    want = rotary_backward(torch.ones_like(x), None, pos, rot)[0]
    assert torch.equal(x.grad, want)
    x.grad = None
    apply_rotary_positions(x, None, pos, rot)[0].float().sum().backward()
    assert torch.equal(x.grad, want)


def test_gradient_against_differences():
    """The map is linear: f(x + h e) - f(x) = h f(e) for any step h.  Powers of
    two and inputs of few bits make x + h e exact; each f is off by half a step
    of its result."""
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    rot = RotaryPositions(32, scaling=WAVE)
    pos = torch.arange(90, 95, device="cuda", dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    x = (torch.randint(-64, 64, (1, 5, 2, 64), generator=g) / 32).half().cuda()
    w = (torch.randint(-64, 64, (1, 5, 2, 64), generator=g) / 32).half().cuda()
    x.requires_grad_()
    dx, = torch.autograd.grad(apply_rotary_positions(x, None, pos, rot)[0], x, w)
    f0 = apply_rotary_positions(x.detach(), None, pos, rot)[0].double()
    for d in (0, 5, 15, 16, 31, 32, 63):
        e = torch.zeros_like(x)
        e[..., d] = 0.5
        f1 = apply_rotary_positions(x.detach() + e, None, pos, rot)[0].double()
        want = ((f1 - f0) * w.double()).sum(-1) / 0.5
        # two columns of a row change; each is under 8 and off by 2^-11 of it,
        # twice, times |w| < 2 over the step 0.5, and dx itself by its rounding
        tol = 2 * 2 * 8 * 2 ** -11 * 2 / 0.5 + 8 * 2 ** -11
        assert (dx[..., d].double() - want).abs().max() <= tol


def test_gradients_of_one_side_and_of_gradients():
    from flash_attn_volta import RotaryPositions, apply_rotary_positions, rotary_backward
    rot = RotaryPositions(64, interleaved=True)
    pos = torch.arange(6, device="cuda")
    q, k = (_inputs(2, 6, 2, 64, torch.float16, s).cuda() for s in (0, 1))
    g = _inputs(2, 6, 2, 64, torch.float16, 2).cuda()
    want = rotary_backward(g, None, pos, rot)[0]
    for a, b in ((q.clone().requires_grad_(), k), (q, k.clone().requires_grad_())):
        qo, ko = apply_rotary_positions(a, b, pos, rot)
        leaf, out = (a, qo) if a.requires_grad else (b, ko)
        got, = torch.autograd.grad(out, leaf, g)
        assert torch.equal(got, want)
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    out = apply_rotary_positions(a, b, pos, rot)[1]          # q's output is not used
    assert torch.autograd.grad(out, (a, b), g, allow_unused=True)[1].equal(want)
    u = g.clone().requires_grad_()
    dx, = torch.autograd.grad(apply_rotary_positions(a, None, pos, rot)[0], a, u, create_graph=True)
    ddu, = torch.autograd.grad(dx, u, q)
    assert torch.equal(ddu, apply_rotary_positions(q, None, pos, rot)[0])


def test_far_positions_keep_their_angles():
    """int64 positions far past where an fp32 angle means anything: the steps are
    exact to 2^-65 turns a position."""
    from fractions import Fraction
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    rot = RotaryPositions(2, base=1.0)                      # one radian a position
    x = torch.zeros((1, 4, 1, 8), dtype=torch.float16, device="cuda")
    x[..., 0] = 1.0
    at = [2 ** 20 + 1, 2 ** 24 + 3, 2 ** 31 + 7, -(2 ** 30)]
    out = apply_rotary_positions(x, None, torch.tensor([at], device="cuda"), rot)[0][0, :, 0, :2]
    two_pi = Fraction("6.28318530717958647692528676655900576839433879875021")
    for i, p in enumerate(at):
        a = float(Fraction(p) % two_pi)
        assert abs(float(out[i, 0]) - np.cos(a)) <= 2 ** -11 + 1e-6
        assert abs(float(out[i, 1]) - np.sin(a)) <= 2 ** -11 + 1e-6


def test_graph_replays_and_other_stream():
    """Replays of a captured forward and backward follow the inputs' and positions'
    contents.  Beside a living eager graph of the same leaves the capture is
    refused (it would end the process), and taken once that is gone."""
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    from flash_attn_volta.forward import FlashAttnArgumentError
    rot = RotaryPositions(128, scaling=YARN)
    q, k = (_inputs(2, 33, h, 128, torch.bfloat16, h).cuda().requires_grad_() for h in (4, 2))
    gq, gk = (_inputs(2, 33, h, 128, torch.bfloat16, 9 + h).cuda() for h in (4, 2))
    pos = torch.arange(33, device="cuda", dtype=torch.int32)

    def step():
        out = apply_rotary_positions(q, k, pos, rot)
        grads = torch.autograd.grad(out, (q, k), (gq, gk))
        return tuple(t.detach() for t in (*out, *grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step()))
    alive = apply_rotary_positions(q, k, pos, rot)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(FlashAttnArgumentError, match="alive"):
        with torch.cuda.graph(g):
            step()
    del alive
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for rep in range(3):
        with torch.no_grad():
            q.mul_(0.5)
            pos.add_(1000)
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_saved_tensor_hooks():
    """What comes back from a hook on saved tensors is read by its own strides."""
    from flash_attn_volta import RotaryPositions, apply_rotary_positions, rotary_backward
    rot = RotaryPositions(32)
    pos = torch.arange(9, device="cuda")[None].expand(2, -1)
    x = _inputs(2, 9, 2, 64, torch.float16, 0).cuda().requires_grad_()
    g = _inputs(2, 9, 2, 64, torch.float16, 1).cuda()
    with torch.autograd.graph.save_on_cpu():
        out = apply_rotary_positions(x, None, pos, rot)[0]
    got, = torch.autograd.grad(out, x, g)
    assert torch.equal(got, rotary_backward(g, None, pos, rot)[0])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[..., :1]):
        out = apply_rotary_positions(x, None, pos, rot)[0]
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(out, x, g)


def test_python_node_gives_the_same(monkeypatch):
    """Without the C++ module the Python Function carries every call."""
    from flash_attn_volta import RotaryPositions, apply_rotary_positions, rotary
    rot = RotaryPositions(32, interleaved=True)
    pos = torch.arange(7, device="cuda")
    q, k = (_inputs(2, 7, h, 64, torch.float16, h).cuda().requires_grad_() for h in (4, 2))
    g = [_inputs(2, 7, h, 64, torch.float16, 5 + h).cuda() for h in (4, 2)]

    def step():
        out = apply_rotary_positions(q, k, pos, rot)
        return (*out, *torch.autograd.grad(out, (q, k), g))

    want = step()
    assert "RotaryFn" in want[0].grad_fn.name() and "_RotaryFn" not in want[0].grad_fn.name()
    monkeypatch.setattr(rotary, "_cpp", None)
    got = step()
    assert "_RotaryFn" in got[0].grad_fn.name()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    u = g[0].clone().requires_grad_()
    a = apply_rotary_positions(q, None, pos, rot)[0]
    dx, = torch.autograd.grad(a, q, u, create_graph=True)
    ddu, = torch.autograd.grad(dx, u, g[0])
    assert torch.equal(ddu, apply_rotary_positions(g[0], None, pos, rot)[0])


def test_empty_and_refused():
    from flash_attn_volta import RotaryPositions, apply_rotary_positions
    from flash_attn_volta.forward import FlashAttnArgumentError
    rot = RotaryPositions(32)
    q = torch.zeros((1, 4, 2, 64), dtype=torch.float16, device="cuda")
    pos = torch.arange(4, device="cuda")
    for shape in ((0, 4, 2, 64), (1, 0, 2, 64), (1, 4, 0, 64)):
        e = torch.zeros(shape, dtype=torch.float16, device="cuda")
        assert apply_rotary_positions(e, e, pos[:shape[1]], rot)[1].shape == shape
    assert apply_rotary_positions(q[:, :, :0], q, pos, rot)[1].equal(q)      # k alone has heads
    assert apply_rotary_positions(q, q[:, :, :0], pos, rot)[0].equal(q)
    for bad in ((q.float(), None, pos, rot), (q, q.bfloat16(), pos, rot), (q, None, pos[:3], rot),
                (q, None, pos.float(), rot), (q, None, pos.cpu(), rot), (q[0], None, pos, rot),
                (q, None, pos, RotaryPositions(128)), (q, None, pos, RotaryPositions(32, device="cpu")),
                (q[..., :60], None, pos, rot), (q, None, pos, None)):
        with pytest.raises(FlashAttnArgumentError):
            apply_rotary_positions(*bad)
