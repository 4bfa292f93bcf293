"""Gated linear recurrence (csrc/gated_scan.cu) against a step-by-step evaluation in 64 bits,
forward, backward and single step.  Bars, max|a-b| / max|b| per output: 16-bit outputs as the
other 16-bit kernels' (one rounding, 2^-11 and 2^-8 relative at most: 1e-3 and 8e-3); 32-bit
ones 2e-5 (a rounding of 2^-25 in a enters once per step of a memory of up to ~10^3 steps)."""
import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from deltagrid_b200.recurrence import GatedRecurrence, gated_scan, gated_scan_packed, gated_scan_step

TOL = {torch.float32: 2e-5, torch.float16: 1e-3, torch.bfloat16: 8e-3}
STATE = 2e-5


def _ref(x, g, o, h0, lengths, resets, dy=None, dh=None):
    """64-bit results by steps: y, h_last and, with dy and dh, the gradients by the formulas."""
    x, g = x.double(), g.double()
    B, T, D = x.shape
    h = h0.double().clone() if h0 is not None else torch.zeros(B, D, dtype=torch.float64, device=x.device)
    n = lengths.long() if lengths is not None else torch.full((B,), T, device=x.device)
    a = torch.sigmoid(g)
    na = torch.sigmoid(-g)
    keep = torch.ones(B, T, 1, dtype=torch.float64, device=x.device)
    if resets is not None:
        keep = (~resets.bool()).double()[..., None]
    sg = torch.sigmoid(o.double()) if o is not None else None
    gate = o.double() * sg if o is not None else torch.ones_like(x)
    y, prev, states = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        live = (t < n)[:, None]
        prev[:, t] = h * keep[:, t]
        new = a[:, t] * prev[:, t] + na[:, t] * x[:, t]
        h = torch.where(live, new, h)
        states[:, t] = h
        y[:, t] = torch.where(live, h * gate[:, t], 0.0)
    if dy is None:
        return y, h
    e = dh.double().clone() if dh is not None else torch.zeros_like(h)
    dx, dg, do = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    dy = dy.double()
    for t in reversed(range(T)):
        live = (t < n)[:, None]
        et = e + dy[:, t] * gate[:, t]
        dx[:, t] = torch.where(live, et * na[:, t], 0.0)
        dg[:, t] = torch.where(live, et * (prev[:, t] - x[:, t]) * a[:, t] * na[:, t], 0.0)
        if o is not None:
            s = sg[:, t]
            do[:, t] = torch.where(live, dy[:, t] * states[:, t] * s * (1 + o[:, t].double() * (1 - s)), 0.0)
        e = torch.where(live, et * a[:, t] * keep[:, t], e)
    return y, h, dx, dg, do, e


def _inputs(B, T, D, dtype, seed, out_gate=True, layout="plain", lengths=None, resets=False, h0=True):
    g = torch.Generator().manual_seed(seed)
    parts = [torch.randn(B, T, D, generator=g), torch.randn(B, T, D, generator=g) * 2 + 2,
             torch.randn(B, T, D, generator=g)]
    parts = [p.to(dtype).cuda() for p in parts]
    if layout == "packed":
        parts = list(torch.cat(parts, -1).split(D, -1))
    elif layout == "time_first":
        parts = [p.transpose(0, 1).contiguous().transpose(0, 1) for p in parts]
    elif layout == "offset":        # rows that start off every vector boundary
        parts = [torch.cat([p[..., :1], p], -1)[..., 1:] for p in parts]
    if not out_gate:
        parts[2] = None
    n = torch.tensor(lengths, dtype=torch.int32).cuda() if lengths is not None else None
    r = (torch.rand(B, T, generator=g) < 0.05).cuda() if resets else None
    h = torch.randn(B, D, generator=g).cuda() if h0 else None
    dy = torch.randn(B, T, D, generator=g).to(dtype).cuda()
    dh = torch.randn(B, D, generator=g).cuda()
    return parts, h, n, r, dy, dh


def _check(parts, h, n, r, dy, dh, dtype, use_dh=True):
    x, gate, o = parts
    leaves = [p.detach().requires_grad_(True) for p in parts if p is not None]
    h_leaf = h.detach().clone().requires_grad_(True) if h is not None else None
    with torch.no_grad():
        y0, l0 = gated_scan(x, gate, o, h, n, r)
    y, last = gated_scan(leaves[0], leaves[1], leaves[2] if o is not None else None, h_leaf, n, r)
    # saving for the backward pass changes nothing (bits: what is padded may be NaN in x alone)
    assert torch.equal(y0, y) and torch.equal(l0, last)
    assert y.dtype == dtype and last.dtype == torch.float32
    want = leaves + ([h_leaf] if h is not None else [])
    outs, gs = ((y, last), (dy, dh)) if use_dh else ((y,), (dy,))
    grads = torch.autograd.grad(outs, want, gs)
    torch.cuda.synchronize()
    ry, rl, rx, rg, ro, rh = _ref(x, gate, o, h, n, r, dy, dh if use_dh else None)
    assert rel_err(y.detach().float().cpu(), ry.cpu()) < TOL[dtype]
    assert rel_err(last.detach().cpu(), rl.cpu()) < STATE
    refs = [rx, rg] + ([ro] if o is not None else []) + ([rh] if h is not None else [])
    for got, ref in zip(grads, refs):
        tol = STATE if got.dtype == torch.float32 else TOL[dtype]
        assert rel_err(got.float().cpu(), ref.cpu()) < tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 2, 3), (3, 127, 64), (1, 128, 66), (2, 129, 130), (2, 700, 40),
                                   (4, 257, 768), (1, 3000, 72)])
def test_forward_and_backward(B, T, D, dtype):
    _check(*_inputs(B, T, D, dtype, seed=T + D), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 5, 1), (3, 70, 7), (2, 300, 65), (1, 2100, 33), (2, 131, 64)])
@pytest.mark.parametrize("start,gap", [(0, 0), (1, 0), (0, 1), (1, 1), (3, 4)])
def test_single_elements_beside_junk(B, T, D, start, gap, dtype):
    """Rows that start at odd and even elements with odd and even strides, NaN before and behind each."""
    (x, g, o), h0, _, r, dy, dh = _inputs(B, T, D, dtype, seed=D + start, resets=True)
    def beside_junk(p):
        wide = torch.full((start + B * T * (D + gap) + 1,), float("nan"), dtype=dtype, device="cuda")
        v = wide[start:start + B * T * (D + gap)].view(B, T, D + gap)[..., :D]
        v.copy_(p)
        return v
    plain = [p.clone().requires_grad_(True) for p in (x, g, o)]
    leaves = [beside_junk(p).requires_grad_(True) for p in (x, g, o)]
    want = gated_scan(*plain, h0, None, r)
    got = gated_scan(*leaves, h0, None, r)
    for a, b in zip(got, _ref(x, g, o, h0, None, r)):
        assert rel_err(a.detach().float().cpu(), b.float().cpu()) < (TOL[dtype] if a.dtype == dtype else STATE)
    want = torch.autograd.grad(want, plain, (dy, dh))
    got = torch.autograd.grad(got, leaves, (beside_junk(dy), dh))
    for a, b in zip(got, want):
        assert rel_err(a.float().cpu(), b.float().cpu()) < TOL[dtype]


@pytest.mark.parametrize("layout", ["packed", "time_first", "offset"])
@pytest.mark.parametrize("D", [64, 65, 96])
def test_strides(layout, D):
    _check(*_inputs(3, 200, D, torch.bfloat16, seed=D, layout=layout, resets=True), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_out_gate_no_h0_no_state_gradient(dtype):
    _check(*_inputs(2, 300, 48, dtype, seed=5, out_gate=False, h0=False), dtype, use_dh=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,lengths", [(140, [0, 140, 1, 128]), (300, [129, 0, 0, 299]), (64, [64, 200, -3, 7]),
                                       (2500, [2500, 1, 1300, 0])])
def test_lengths_with_anything_in_the_padding(T, lengths, dtype):
    parts, h, n, r, dy, dh = _inputs(4, T, 40, dtype, seed=T, lengths=lengths, resets=True)
    n_c = n.clamp(0, T)
    clean = _ref(*[p.clone() for p in parts], h, n_c, r, dy, dh)
    pad = torch.arange(T, device="cuda")[None] >= n_c[:, None]
    for i, junk in enumerate((float("nan"), float("inf"), float("-inf"))):
        parts[i][pad] = junk
    dy[pad] = float("nan")
    leaves = [p.detach().requires_grad_(True) for p in parts]
    h_leaf = h.clone().requires_grad_(True)
    y, last = gated_scan(*leaves, h_leaf, n, r)
    grads = torch.autograd.grad((y, last), [*leaves, h_leaf], (dy, dh))
    torch.cuda.synchronize()
    assert not y[pad].any() and not any(g[pad].any() for g in grads[:3])
    for got, ref in zip((y, last, *grads), clean):
        tol = STATE if got.dtype == torch.float32 else TOL[dtype]
        assert rel_err(got.detach().float().cpu(), ref.cpu()) < tol
    assert torch.equal(last[n_c == 0], h[n_c == 0])          # an empty row hands its state on
    assert torch.equal(grads[3][n_c == 0], dh[n_c == 0])


def test_lengths_int64_and_resets_everywhere():
    parts, h, _, _, dy, dh = _inputs(2, 90, 32, torch.float32, seed=8)
    n = torch.tensor([90, 2 ** 40], dtype=torch.int64, device="cuda")
    r = torch.ones(2, 90, dtype=torch.uint8, device="cuda")
    y, last = gated_scan(*parts, h, n, r)
    ry, rl = _ref(*parts, h, None, r)
    assert rel_err(y.cpu(), ry.cpu()) < STATE and rel_err(last.cpu(), rl.cpu()) < STATE


def test_extreme_gates_stay_finite():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 260, 32, generator=g).cuda()
    gate = (torch.randint(-1, 2, (2, 260, 32), generator=g) * 3e4).float().cuda()
    o = (torch.randint(-1, 2, (2, 260, 32), generator=g) * 3e4).float().cuda()
    dy = torch.randn(2, 260, 32, generator=g).cuda()
    leaves = [t.requires_grad_(True) for t in (x, gate, o)]
    y, last = gated_scan(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    ry, rl, rx, rg, ro, _ = _ref(x.detach(), gate.detach(), o.detach(), None, None, None, dy, None)
    for got, ref in zip((y, last, *grads), (ry, rl, rx, rg, ro)):
        assert torch.isfinite(got).all()
        assert float((got.detach().double() - ref).abs().max()) <= 2e-5 * max(1.0, float(ref.abs().max()))


@pytest.mark.parametrize("out_gate", [True, False])
def test_packed_equals_parts(out_gate):
    parts, h, _, r, dy, dh = _inputs(2, 150, 40, torch.bfloat16, seed=3, resets=True, out_gate=out_gate)
    live = [p for p in parts if p is not None]
    packed = torch.cat(live, -1).requires_grad_(True)
    y, last = gated_scan_packed(packed, h, None, r, out_gate=out_gate)
    (gp,) = torch.autograd.grad((y, last), [packed], (dy, dh))
    leaves = [p.detach().requires_grad_(True) for p in live]
    y2, last2 = gated_scan(*leaves, *([None] if not out_gate else []), h, None, r)
    gs = torch.autograd.grad((y2, last2), leaves, (dy, dh))
    assert torch.equal(y, y2) and torch.equal(last, last2) and torch.equal(gp, torch.cat(gs, -1))


def test_gradients_against_differences():
    """Central differences of the forward pass itself: a loss of smooth 32-bit values, step 1e-2,
    so about 1e-4 of curvature and 1e-5 of rounding against directional slopes of order 1."""
    parts, h, n, r, dy, dh = _inputs(2, 130, 24, torch.float32, seed=9, lengths=[130, 77], resets=True)
    leaves = [p.detach().requires_grad_(True) for p in parts] + [h.clone().requires_grad_(True)]

    def loss(ts):
        y, last = gated_scan(*ts, n, r)
        return (y.double() * dy).sum() + (last.double() * dh).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i in range(4):
        v = torch.randn(leaves[i].shape, generator=gen).cuda()
        v = v / v.norm()
        ts = [t.detach() for t in leaves]
        up, dn = list(ts), list(ts)
        up[i], dn[i] = ts[i] + 1e-2 * v, ts[i] - 1e-2 * v
        slope = float((loss(up) - loss(dn)) / 2e-2)
        want = float((grads[i].double() * v).sum())
        assert abs(slope - want) < 5e-3 * max(1.0, float(grads[i].double().norm()) / 10), (i, slope, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,D", [(1, 1), (5, 33), (256, 768), (3, 130)])
def test_step_continues_a_sequence(B, D, dtype):
    parts, h, _, _, _, _ = _inputs(B, 3, D, dtype, seed=B + D, layout="packed")
    y, last = gated_scan(*parts, h)
    s = h.clone()
    outs = [gated_scan_step(parts[0][:, t], parts[1][:, t], s, parts[2][:, t]) for t in range(3)]
    ry, rl = _ref(*parts, h, None, None)
    assert rel_err(s.cpu(), rl.cpu()) < STATE and rel_err(last.cpu(), rl.cpu()) < STATE
    assert rel_err(torch.stack(outs, 1).float().cpu(), ry.cpu()) < TOL[dtype]
    s2 = h.clone()
    assert rel_err(gated_scan_step(parts[0][:, 0], parts[1][:, 0], s2).float().cpu(),
                   _ref(parts[0][:, :1], parts[1][:, :1], None, h, None, None)[0][:, 0].cpu()) < TOL[dtype]


def test_empty_sizes():
    h = torch.randn(2, 8, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    y, last = gated_scan(x, x.detach(), x.detach(), h)
    assert y.shape == (2, 0, 8) and torch.equal(last, h)
    (gh,) = torch.autograd.grad(last, [h], torch.ones_like(last))
    assert torch.equal(gh, torch.ones_like(h))
    z = torch.zeros(0, 5, 8, device="cuda")
    y, last = gated_scan(z, z)
    assert y.shape == (0, 5, 8) and last.shape == (0, 8)


def test_results_repeat_and_run_on_a_side_stream():
    parts, h, _, r, dy, dh = _inputs(2, 2000, 64, torch.bfloat16, seed=4, resets=True)
    leaves = [p.detach().requires_grad_(True) for p in parts]
    y, last = gated_scan(*leaves, h, None, r)
    g1 = torch.autograd.grad((y, last), leaves, (dy, dh))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2, last2 = gated_scan(*leaves, h, None, r)
        g2 = torch.autograd.grad((y2, last2), leaves, (dy, dh))
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(last, last2) and all(torch.equal(a, b) for a, b in zip(g1, g2))


def test_layer_step_equals_forward():
    torch.manual_seed(0)
    m = GatedRecurrence(48).cuda()
    x = torch.randn(3, 6, 48, device="cuda")
    with torch.no_grad():
        y, s = m(x)
        st, outs = None, []
        for t in range(6):
            o, st = m.step(x[:, t:t + 1], st)
            outs.append(o)
    assert rel_err(torch.cat(outs, 1).cpu(), y.cpu()) < 1e-4 and rel_err(st.cpu(), s.cpu()) < 1e-4


def test_refusals():
    x = torch.zeros(2, 4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        gated_scan(x.cpu(), x.cpu())
    with pytest.raises(RuntimeError, match="x's shape"):
        gated_scan(x, x[:, :3])
    with pytest.raises(RuntimeError, match="dtype"):
        gated_scan(x, x.half())
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        gated_scan(x.double(), x.double())
    with pytest.raises(RuntimeError, match="h0"):
        gated_scan(x, x, h0=torch.zeros(2, 8, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError, match="lengths"):
        gated_scan(x, x, lengths=torch.zeros(3, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="resets"):
        gated_scan(x, x, resets=torch.zeros(2, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="packed"):
        gated_scan_packed(torch.zeros(2, 4, 10, device="cuda"))
    with pytest.raises(RuntimeError, match="in place"):
        gated_scan_step(x[:, 0], x[:, 0], torch.zeros(2, 8, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no backward"):
        gated_scan_step(x[:, 0].clone().requires_grad_(True), x[:, 0], torch.zeros(2, 8, device="cuda"))
    leaf = x.clone().requires_grad_(True)
    y, _ = gated_scan(leaf, x)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_wait_timeout_flags_status():
    """Wait budget zero: the exchange between the CTAs of a cluster gives up at once, the launch says
    so and ends; the next call is right again."""
    from deltagrid_b200 import hsru_delta_cuda as ext
    parts, h, _, _, _, _ = _inputs(1, 4000, 64, torch.bfloat16, seed=21)       # few channels: clusters
    want = gated_scan(*parts, h)
    torch.cuda.synchronize()
    ext.device_status()
    old = ext.set_wait_limit(0)
    try:
        gated_scan(*parts, h)
        torch.cuda.synchronize()
    finally:
        ext.set_wait_limit(old)
    assert ext.device_status() & 0x4
    again = gated_scan(*parts, h)
    torch.cuda.synchronize()
    assert ext.device_status() == 0
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_output_gates_down_to_the_lowest_value(dtype):
    """z sigmoid(z) and its slope vanish for very negative z, masks of the type's lowest value among them."""
    parts, h, _, _, dy, dh = _inputs(2, 300, 40, dtype, seed=31)
    low = torch.finfo(dtype).min
    closed = torch.tensor([low, low / 2, -1e30, -1e20, -1e5, -120.0, -90.0, -88.0, -60.0], device="cuda").to(dtype)
    parts[2][:, ::3] = closed[torch.arange(100 * 40, device="cuda") % 9].view(100, 40)
    _check(parts, h, None, None, dy, dh, dtype)
    s = h.clone()
    y = gated_scan_step(parts[0][:, 0], parts[1][:, 0], s, parts[2][:, 0])
    want = _ref(*[p[:, :1] for p in parts], h, None, None)[0][:, 0]
    assert rel_err(y.float().cpu(), want.cpu()) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,t", [(2, 300, 64, 137), (1, 3000, 72, 1700), (2, 40, 33, 0), (3, 700, 130, 699)])
def test_a_gate_that_is_not_a_number_shows(B, T, D, t, dtype):
    """The outputs and gradients that the formulas make NaN, and no others."""
    parts, h, _, r, dy, dh = _inputs(B, T, D, dtype, seed=t)
    parts[1][0, t, 5] = float("nan")
    leaves = [p.detach().requires_grad_(True) for p in parts] + [h.clone().requires_grad_(True)]
    y, last = gated_scan(*leaves, None, r)
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    for got, ref in zip((y, last, *grads), _ref(*parts, h, None, r, dy, dh)):
        bad = torch.isnan(ref)
        assert torch.equal(torch.isnan(got), bad)
        tol = STATE if got.dtype == torch.float32 else TOL[dtype]
        assert rel_err(got.detach().float().masked_fill(bad, 0.0).cpu(), ref.masked_fill(bad, 0.0).cpu()) < tol
    s = h.clone()
    y = gated_scan_step(parts[0][:, t], parts[1][:, t], s, parts[2][:, t])
    assert torch.isnan(y[0, 5]) and torch.isnan(s[0, 5]) and int(torch.isnan(y).sum() + torch.isnan(s).sum()) == 2


def test_closed_gates_forget_any_state():
    """sigmoid of a very negative gate is 0 to a state of any finite size."""
    h = torch.full((2, 40), 3e38, device="cuda")
    x = torch.randn(2, 3, 40, generator=torch.Generator().manual_seed(1)).cuda()
    gate = torch.full_like(x, -1e4)
    gate[0, :, ::2], gate[1, :, ::2] = torch.finfo(torch.float32).min, float("-inf")
    y, last = gated_scan(x, gate, None, h)
    assert rel_err(y.cpu(), x.cpu()) < STATE and rel_err(last.cpu(), x[:, -1].cpu()) < STATE
    s = h.clone()
    assert rel_err(gated_scan_step(x[:, 0], gate[:, 0], s).cpu(), x[:, 0].cpu()) < STATE


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,t", [(2, 300, 64, 137), (1, 3000, 72, 1700), (4, 600, 768, 33), (2, 90, 33, 64),
                                     (8, 2100, 64, 2050), (64, 40, 130, 8)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_nothing_crosses_a_reset(B, T, D, t, junk, dtype):
    """A state that is not finite stays in its document, and so does a gradient."""
    parts, h, _, _, dy, dh = _inputs(B, T, D, dtype, seed=T + t)
    r = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    r[:, t] = True
    if t > 40:
        r[:, [5, t - 1]] = True          # several in a thread's steps and in a warp's
    cut = lambda ts, a, b: [p[:, a:b] for p in ts]  # noqa: E731
    zero = torch.zeros_like(h)
    # forward: the document that starts at t
    sick = [p.clone() for p in parts]
    sick[0][:, t - 1] = junk
    sick_h = torch.full_like(h, junk)
    leaves = [p.requires_grad_(True) for p in sick] + [sick_h.requires_grad_(True)]
    y, last = gated_scan(*leaves, None, r)
    ry, rl, rx, rg, ro, _ = _ref(*cut(parts, t, T), zero, None, None, dy[:, t:], dh)
    grads = torch.autograd.grad((y, last), leaves, (dy, dh))
    for got, ref in zip((y[:, t:], last, *cut(grads[:3], t, T)), (ry, rl, rx, rg, ro)):
        tol = STATE if got.dtype == torch.float32 else TOL[dtype]
        assert rel_err(got.detach().float().cpu(), ref.cpu()) < tol
    # backward: the documents before it
    leaves = [p.detach().requires_grad_(True) for p in parts] + [h.clone().requires_grad_(True)]
    y, last = gated_scan(*leaves, None, r)
    sick_dy = dy.clone()
    sick_dy[:, t] = junk
    grads = torch.autograd.grad((y, last), leaves, (sick_dy, torch.full_like(dh, junk)))
    refs = _ref(*cut(parts, 0, t), h, None, r[:, :t], dy[:, :t], zero)[2:]
    for got, ref in zip((*cut(grads[:3], 0, t), grads[3]), refs):
        tol = STATE if got.dtype == torch.float32 else TOL[dtype]
        assert rel_err(got.float().cpu(), ref.cpu()) < tol


def test_a_reset_at_the_first_step_drops_h0():
    parts, _, _, _, dy, dh = _inputs(3, 50, 40, torch.float32, seed=4)
    h = torch.full((3, 40), float("nan"), device="cuda", requires_grad=True)
    r = torch.zeros(3, 50, dtype=torch.bool, device="cuda")
    r[:, 0] = True
    y, last = gated_scan(*parts, h, None, r)
    want, rl = _ref(*parts, None, None, None)
    assert rel_err(y.detach().cpu(), want.cpu()) < STATE and rel_err(last.detach().cpu(), rl.cpu()) < STATE
    (g,) = torch.autograd.grad((y, last), [h], (dy, dh))
    assert not g.any()


def test_an_infinite_state_stays_where_nothing_drops_it():
    """Products of many small gates vanish in 32 bits; that is not a reset."""
    x = torch.zeros(2, 600, 64, device="cuda")
    x[:, 3] = float("inf")
    gate = torch.full_like(x, -20.0)
    r = torch.zeros(2, 600, dtype=torch.bool, device="cuda")
    r[:, 2] = True
    for resets in (None, r):
        y, last = gated_scan(x, gate, None, None, None, resets)
        assert not torch.isfinite(y[:, 3:]).any() and not torch.isfinite(last).any() and torch.isfinite(y[:, :3]).all()


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x = torch.randn(2, 5, 8, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_scan(d, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_scan(x, x, None, fwd.make_dual(x[:, 0].clone(), x[:, 0].clone()))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_scan_packed(fwd.make_dual(torch.zeros(2, 5, 24, device="cuda"), torch.ones(2, 5, 24, device="cuda")))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_scan_step(d[:, 0], x[:, 0], torch.zeros(2, 8, device="cuda"))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            gated_scan(d, x)
    gated_scan(x, x)


def test_step_counts_as_a_change_of_the_state():
    """A state that autograd has saved and a step has advanced since is an error in the backward pass."""
    w = torch.randn(2, 8, device="cuda", requires_grad=True)
    state = w * 2.0
    loss = state.pow(2).sum()
    with torch.no_grad():
        gated_scan_step(torch.zeros(2, 8, device="cuda"), torch.zeros(2, 8, device="cuda"), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        s = torch.ones(2, 8, device="cuda")
        gated_scan_step(torch.zeros(2, 8, device="cuda"), torch.zeros(2, 8, device="cuda"), s)
    assert float(s.sum()) == 8.0


def test_step_of_very_many_rows():
    g = torch.Generator(device="cuda").manual_seed(2)
    x, gate = (torch.randn(70001, 3, generator=g, device="cuda").half() for _ in range(2))
    h = torch.randn(70001, 3, generator=g, device="cuda")
    want = _ref(x[:, None], gate[:, None], None, h, None, None)[1]
    y = gated_scan_step(x, gate, h)
    assert rel_err(h.cpu(), want.cpu()) < STATE and rel_err(y.float().cpu(), want.cpu()) < TOL[torch.float16]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,D", [(2, 300, 514), (40, 400, 66), (3, 1100, 1026)])
def test_pairs_of_channels_without_wide_copies(B, T, D, dtype):
    _check(*_inputs(B, T, D, dtype, seed=B, resets=True), dtype)


@pytest.mark.parametrize("B,T,D", [(100, 600, 512), (33, 1500, 520)])
def test_more_than_one_wave(B, T, D):
    _check(*_inputs(B, T, D, torch.bfloat16, seed=B, resets=True), torch.bfloat16)
