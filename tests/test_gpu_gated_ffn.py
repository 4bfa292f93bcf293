"""Gated feed-forward block (csrc/gated_ffn*.cu) against its formulas in 64 bits.  Bars,
max|a-b| / max|b|: the forward pass rounds once (2^-11 and 2^-8 relative at most: 1e-3 for
f16, 8e-3 for bf16, as the other 16-bit kernels' tests); the gradients of x and the weights
pass through dG and dU rounded to the storage type as well: twice that.  f32 is held to 1e-5
(sums of up to 2 x 10^3 products in 32 bits)."""
import math

import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from deltagrid_b200 import hsru_delta_cuda as ext
    from deltagrid_b200.ffn import GatedFFN, gated_ffn

TOL = {torch.float32: 1e-5, torch.float16: 1e-3, torch.bfloat16: 8e-3}


def _act(z, kind):
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def _ref(x, w, b, kind, dh=None):
    x, w = x.double(), w.double()
    z = x @ w.T + (b.double() if b is not None else 0.0)
    F = w.shape[0] // 2
    g, u = z[..., :F], z[..., F:]
    f, df = _act(g, kind)
    if dh is None:
        return f * u
    d = dh.double()
    dz = torch.cat([d * u * df, d * f], -1)
    return f * u, dz @ w, dz.T @ x, dz.sum(0)


def _inputs(M, D, F, dtype, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, D, generator=g).to(dtype).cuda()
    w = (torch.randn(2 * F, D, generator=g) / math.sqrt(D)).to(dtype).cuda()
    b = (torch.randn(2 * F, generator=g) * 0.3).to(dtype).cuda() if bias else None
    dh = torch.randn(M, F, generator=g).to(dtype).cuda()
    return x, w, b, dh


def _check(x, w, b, dh, kind):
    tol = TOL[x.dtype]
    with torch.no_grad():
        h0 = gated_ffn(x, w, b, kind)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    h = gated_ffn(*leaves, *([None] if b is None else []), kind)
    assert torch.equal(h0, h)
    grads = torch.autograd.grad(h, leaves, dh)
    torch.cuda.synchronize()
    rh, rx, rw, rb = _ref(x, w, b, kind, dh)
    assert rel_err(h.detach().float().cpu(), rh.cpu()) < tol
    assert rel_err(grads[0].float().cpu(), rx.cpu()) < 2 * tol
    assert rel_err(grads[1].float().cpu(), rw.cpu()) < 2 * tol
    if b is not None:
        assert rel_err(grads[2].float().cpu(), rb.cpu()) < tol
    assert ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,D,F", [(1, 8, 8), (2, 24, 40), (13, 64, 72), (17, 100, 130), (129, 328, 264), (300, 7, 5),
                                   (1000, 512, 640), (257, 768, 768), (40, 2048, 64), (520, 64, 1032)])
def test_forward_and_backward(M, D, F, dtype):
    _check(*_inputs(M, D, F, dtype, seed=M + D + F), "silu")


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("M,D,F", [(2600, 136, 760), (2560, 768, 768), (9000, 72, 1104), (300, 192, 4096)])
def test_many_tiles(M, D, F, bias):
    """Tiles of 128 features and of 64, several to a CTA, the last ones ragged."""
    x, w, b, dh = _inputs(M, D, F, torch.bfloat16, seed=M, bias=bias)
    _check(x, w, b, dh, "silu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [3, 130, 700])
def test_gelu_without_bias(M, dtype):
    _check(*_inputs(M, 256, 384, dtype, seed=M, bias=False), "gelu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128])
@pytest.mark.parametrize("D,F", [(768, 768), (136, 88), (1096, 520)])
def test_few_tokens(M, D, F, dtype):
    x, w, b, _ = _inputs(M, D, F, dtype, seed=M)
    h = gated_ffn(x, w, b)
    torch.cuda.synchronize()
    assert rel_err(h.float().cpu(), _ref(x, w, b, "silu").cpu()) < TOL[dtype]
    assert ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,F", [(9, 4096, 128), (16, 2056, 1000), (33, 64, 40), (47, 200, 4000), (64, 8, 8),
                                   (97, 4096, 136), (128, 512, 9480), (129, 1536, 72), (200, 4104, 1000),
                                   (255, 1544, 4096), (256, 1536, 520), (256, 1528, 520), (257, 2048, 64),
                                   (7, 4096, 4104)])
def test_tokens_against_a_split_axis(M, D, F, act, dtype):
    """Up to 256 tokens: parts of D on several CTAs, tails of D, F and the tokens, one part and eight."""
    x, w, b, _ = _inputs(M, D, F, dtype, seed=M + F)
    h = gated_ffn(x, w, b, act)
    torch.cuda.synchronize()
    assert rel_err(h.float().cpu(), _ref(x, w, b, act).cpu()) < TOL[dtype]
    assert torch.equal(h, gated_ffn(x, w, b, act))
    assert ext.device_status() == 0


@pytest.mark.parametrize("M", [5, 200])
@pytest.mark.parametrize("D,F,off", [(64, 64, 0), (64, 64, 1), (72, 40, 4), (72, 40, 8), (65, 33, 3)])
def test_row_strides_and_offsets(M, D, F, off):
    """x and dh as column slices of wider tensors: rows that start on and off vector boundaries."""
    x, w, b, dh = _inputs(M, D, F, torch.bfloat16, seed=off)
    wide_x = torch.zeros(M, D + 24, dtype=x.dtype, device="cuda")
    wide_x[:, off:off + D] = x
    wide_h = torch.zeros(M, F + 24, dtype=x.dtype, device="cuda")
    wide_h[:, off:off + F] = dh
    _check(wide_x[:, off:off + D], w, b, wide_h[:, off:off + F], "silu")


def test_offset_weights():
    """Weights and bias that start off every vector boundary."""
    x, w, b, dh = _inputs(150, 96, 64, torch.float16, seed=2)
    wo = torch.cat([w.flatten()[:1], w.flatten()])[1:].view_as(w)
    bo = torch.cat([b[:3], b])[3:]
    _check(x, wo, bo, dh, "silu")


def test_leading_dimensions_broadcast_rows_and_layer():
    torch.manual_seed(1)
    m = GatedFFN(64, 96).cuda().half()
    x = torch.randn(3, 5, 64, device="cuda").half()
    with torch.no_grad():
        y = m(x)
    h = _ref(x.view(15, 64), m.fc1.weight, m.fc1.bias, "silu")
    want = h @ m.fc2.weight.double().T + m.fc2.bias.double()
    assert y.shape == (3, 5, 64) and rel_err(y.view(15, 64).detach().float().cpu(), want.detach().cpu()) < 2e-3
    one = torch.randn(1, 64, device="cuda").half().expand(7, 64)      # row stride 0
    h = gated_ffn(one, m.fc1.weight.detach())
    assert rel_err(h.float().cpu(), _ref(one, m.fc1.weight.detach(), None, "silu").cpu()) < 1e-3
    h = gated_ffn(x[0, 0], m.fc1.weight.detach())                     # one vector
    assert h.shape == (96,)


def test_no_rows_and_partial_gradients():
    w = torch.randn(32, 16, device="cuda").half().requires_grad_(True)
    b = torch.randn(32, device="cuda").half().requires_grad_(True)
    x = torch.zeros(0, 16, device="cuda").half().requires_grad_(True)
    h = gated_ffn(x, w, b)
    assert h.shape == (0, 16)
    gx, gw, gb = torch.autograd.grad(h, [x, w, b], torch.zeros_like(h))
    assert gx.shape == (0, 16) and not gw.any() and not gb.any()
    x, w, b, dh = _inputs(140, 128, 64, torch.bfloat16, seed=6)
    rh, rx, rw, rb = _ref(x, w, b, "silu", dh)
    for i, ref in enumerate((rx, rw, rb)):
        leaves = [x, w, b]
        leaves[i] = leaves[i].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(gated_ffn(*leaves), [leaves[i]], dh)
        assert rel_err(g.float().cpu(), ref.cpu()) < 2 * TOL[torch.bfloat16]


def test_large_values_saturate_as_the_formula_does():
    """Gates of both signs and every size up to f16's largest finite products."""
    x = torch.tensor([[1.0, 0.0] * 4, [-1.0, 0.0] * 4], device="cuda").half().repeat(70, 1)
    w = torch.zeros(64, 8, device="cuda").half()
    w[:32, 0] = torch.linspace(-2000, 2000, 32).half().cuda()
    w[32:, 0] = 1.0
    h = gated_ffn(x, w)
    ref = _ref(x, w, None, "silu")
    assert torch.isfinite(h).all() and rel_err(h.float().cpu(), ref.cpu()) < 1e-3


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gradients_against_differences(kind):
    """Central differences of the 32-bit forward pass, step 1e-2 along unit directions: curvature
    of about 1e-4 and rounding of about 1e-5 against slopes of the gradients' size."""
    x, w, b, dh = _inputs(33, 40, 24, torch.float32, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def loss(ts):
        return (gated_ffn(*ts, kind).double() * dh).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=gen).cuda()
        v = v / v.norm()
        ts = [t.detach() for t in leaves]
        up, dn = list(ts), list(ts)
        up[i], dn[i] = ts[i] + 1e-2 * v, ts[i] - 1e-2 * v
        slope = float((loss(up) - loss(dn)) / 2e-2)
        assert abs(slope - float((grads[i].double() * v).sum())) < 5e-3 * max(1.0, float(grads[i].norm()) / 10)


def test_results_repeat_and_run_on_a_side_stream():
    x, w, b, dh = _inputs(1500, 512, 384, torch.bfloat16, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    g1 = torch.autograd.grad(gated_ffn(*leaves), leaves, dh)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g2 = torch.autograd.grad(gated_ffn(*leaves), leaves, dh)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(g1, g2))


def test_refusals():
    x = torch.zeros(4, 16, device="cuda").half()
    w = torch.zeros(24, 16, device="cuda").half()
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, w, activation="relu")
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        gated_ffn(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="dtype"):
        gated_ffn(x, w.float())
    with pytest.raises(RuntimeError, match="expected x"):
        gated_ffn(x, w[:, :8])
    with pytest.raises(RuntimeError, match="expected x"):
        gated_ffn(x, w[:23])
    with pytest.raises(RuntimeError, match="bias"):
        gated_ffn(x, w, torch.zeros(12, device="cuda").half())
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        gated_ffn(x.double(), w.double())
    leaf = w.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(gated_ffn(x, leaf).sum(), leaf, create_graph=True)


def test_wait_timeout_flags_status():
    """Wait budget zero: the kernel's first waits give up, it drains what it issued, flags
    DG_DEVCHK_TIMEOUT and returns; the next call is right again."""
    x, w, b, dh = _inputs(600, 256, 384, torch.bfloat16, seed=8)
    want = gated_ffn(x, w, b)
    torch.cuda.synchronize()
    ext.device_status()
    old = ext.set_wait_limit(0)
    try:
        gated_ffn(x, w, b)
        torch.cuda.synchronize()
    finally:
        ext.set_wait_limit(old)
    assert ext.device_status() & 0x4
    again = gated_ffn(x, w, b)
    torch.cuda.synchronize()
    assert ext.device_status() == 0 and torch.equal(want, again)


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,dtype", [(4, 16, torch.bfloat16), (100, 16, torch.bfloat16), (600, 16, torch.bfloat16),
                                       (70, 15, torch.bfloat16), (70, 16, torch.float32)])
def test_very_negative_gates(M, D, dtype, kind):
    """Both activations and their slopes vanish down to the type's lowest value."""
    x = torch.zeros(M, D, device="cuda", dtype=dtype)
    x[:, 0] = 1.0
    low = torch.finfo(dtype).min
    z = torch.tensor([low, low / 2, -1e38, -1e30, -1e20, -1e12, -1e5, -120.0, -90.0, -88.0, -60.0, -13.0, -5.0, -0.5,
                      0.0, 0.5, 5.0, 13.0, 60.0], device="cuda")
    w = torch.zeros(64, D, device="cuda", dtype=dtype)
    w[:32, 0] = z[torch.arange(32) % 19].to(dtype)
    w[32:, 0] = 1.0
    dh = torch.randn(M, 32, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    h = gated_ffn(*leaves, None, kind)
    grads = torch.autograd.grad(h, leaves, dh)
    for i, (got, ref) in enumerate(zip((h, *grads), _ref(x.detach(), w.detach(), None, kind, dh))):
        assert rel_err(got.detach().float().cpu(), ref.cpu()) < TOL[dtype] * (1 if i == 0 else 2)


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_very_positive_gates(kind):
    """Slopes of 1 up to the largest values; f(z) = z."""
    z = torch.tensor([13.0, 100.0, 1e4, 1e12, 1e20, 1e30, 3e38, 2.0], device="cuda")
    w = torch.zeros(16, 8, device="cuda")
    w[:8, 0], w[8:, 0] = z, 1.0
    x = torch.zeros(1, 8, device="cuda")
    x[:, 0] = 1.0
    w.requires_grad_(True)
    h = gated_ffn(x, w, None, kind)
    (g,) = torch.autograd.grad(h, [w], torch.ones_like(h))
    rh, _, rw, _ = _ref(x, w.detach(), None, kind, torch.ones_like(h))
    for got, ref in ((h, rh), (g, rw)):
        assert float(((got.detach().double() - ref).abs() / ref.abs().clamp(min=1e-30)).max()) < 1e-5


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x, w, b, _ = _inputs(4, 16, 8, torch.float16, seed=1)
    with fwd.dual_level():
        for i in range(3):
            a = [x, w, b]
            a[i] = fwd.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                gated_ffn(*a)


def test_autocast_runs_in_its_type():
    x, w, b, dh = _inputs(40, 64, 48, torch.float32, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = gated_ffn(*leaves)
        mixed = gated_ffn(x.bfloat16(), w, b)
    assert h.dtype == torch.bfloat16 and torch.equal(h, mixed)
    grads = torch.autograd.grad(h, leaves, dh.bfloat16())
    low = [t.bfloat16() for t in (x, w, b)]
    assert torch.equal(h, gated_ffn(*low))
    for got, ref in zip((h, *grads), _ref(*low, "silu", dh.bfloat16())):
        assert rel_err(got.detach().float().cpu(), ref.cpu()) < 2 * TOL[torch.bfloat16]
    assert all(g.dtype == torch.float32 for g in grads)
    m = GatedFFN(64, 48).cuda()
    with torch.autocast("cuda", dtype=torch.float16):
        assert m(torch.nn.functional.layer_norm(x, (64,))).dtype == torch.float16
        with torch.autocast("cuda", enabled=False):
            assert gated_ffn(x, w).dtype == torch.float32


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,dtype", [(4, 16, torch.bfloat16), (100, 16, torch.float16), (600, 16, torch.bfloat16),
                                       (70, 15, torch.bfloat16), (70, 16, torch.float32)])
def test_what_is_not_a_number_shows(M, D, dtype, kind):
    """A NaN in a row of x, in its outputs and gradients; no other row's."""
    x, w, b, dh = _inputs(M, D, 32, dtype, seed=M)
    x[2, 3] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    h = gated_ffn(*leaves, kind)
    gx, gw, gb = torch.autograd.grad(h, leaves, dh)
    rows = torch.arange(M, device="cuda") == 2
    assert torch.equal(torch.isnan(h).all(1), rows) and torch.equal(torch.isnan(h).any(1), rows)
    assert torch.equal(torch.isnan(gx).all(1), rows) and torch.equal(torch.isnan(gx).any(1), rows)
    assert torch.isnan(gw).all() and torch.isnan(gb).all()
