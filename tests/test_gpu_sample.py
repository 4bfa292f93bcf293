"""Token sampling (csrc/sample.cu) against its definition.  Tokens have to be equal to an
evaluation in Python integers over the masses floor(2^40 exp((l - max) / T)), whose
exponentials are torch's in 32 bits as the operator's are.  Against 64-bit probabilities the
log-probability is held to 1e-5 (masses carry 2^-24, their sums less)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from deltagrid_b200.sampling import sample

ONE = 1 << 40


def _kept(l, T, k, p, m):
    """The kept masses of one row (a list of Python integers) by the definition."""
    l = l.float()
    l = torch.where(torch.isnan(l), float("-inf"), l) + 0.0
    V = l.numel()
    top = l.max()
    greedy = not T > 0
    z = (l - top) / torch.tensor(1.0 if greedy else T, dtype=torch.float32, device=l.device)
    w = (torch.exp(z).double() * ONE).floor()
    w = torch.where(l == top, float(ONE), w)
    w = [int(v) for v in torch.where(torch.isneginf(l) | torch.isnan(w), 0.0, w).tolist()]
    if math.isinf(float(top)) and float(top) < 0:
        return [0] * V
    vals = l.tolist()
    order = sorted(range(V), key=lambda i: (-vals[i], i))
    k = 1 if greedy else (V if k <= 0 or k > V else k)
    order = order[:k]
    total = sum(w[i] for i in order)
    P = int(min(max(float(torch.tensor(p, dtype=torch.float32)), 0.0), 1.0) * (1 << 24))
    tau = max(1, -((-P * total) >> 24))
    least = int(float(torch.tensor(min(max(m, 0.0), 1.0), dtype=torch.float32)) * ONE)
    kept, before = [0] * V, 0
    for i in order:
        if before >= tau:
            break
        before += w[i]
        if w[i] >= least:
            kept[i] = w[i]
    return kept


def _draw(kept, u):
    total = sum(kept)
    if total == 0:
        return -1, -math.inf
    at = (int(u * (1 << 24)) * total) >> 24
    run = 0
    for i, w in enumerate(kept):
        run += w
        if run > at:
            return i, math.log(w / total)


def _check(logits, u, T=1.0, k=0, p=1.0, m=0.0):
    token, logprob = sample(logits, u, T, k, p, m)
    torch.cuda.synchronize()
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for i in range(logits.shape[0]):
        want, lp = _draw(_kept(logits[i], at(T, i), at(k, i), at(p, i), at(m, i)), u[i].item())
        assert token[i].item() == want, (i, token[i].item(), want)
        assert logprob[i].item() == lp or abs(logprob[i].item() - lp) < 1e-5 * max(1.0, abs(lp))


def _logits(B, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    u = torch.randint(0, 1 << 24, (B,), generator=g).float() / (1 << 24)
    return (torch.randn(B, V, generator=g) * scale).to(dtype).cuda(), u.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4099, 32000])
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 40, 0.95, 0.05),
                                     (0.0, 5, 0.5, 0.0), (100.0, 0, 0.99, 0.0)])
def test_tokens_equal_the_definition(V, T, k, p, m, dtype):
    logits, u = _logits(6 if V < 30000 else 3, V, dtype, seed=V + k)
    _check(logits, u, T, k, p, m)


@pytest.mark.parametrize("V", [70001, 150000])
def test_large_vocabularies(V):
    for dtype in (torch.float32, torch.bfloat16):
        logits, u = _logits(2, V, dtype, seed=V)
        _check(logits, u, 0.9, 0, 0.92, 0.0)
        _check(logits, u, 1.1, 300, 0.9, 0.001)


def test_parameters_per_row():
    B = 40
    logits, u = _logits(B, 2000, torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(6)
    T = (torch.rand(B, generator=g) * 2).cuda()
    T[3] = 0.0
    k = torch.randint(-5, 100, (B,), generator=g).cuda()             # int64: converted
    p = torch.rand(B, generator=g).cuda()
    m = (torch.rand(B, generator=g) * 0.2).cuda()
    _check(logits, u, T, k, p, m)
    _check(logits, u, T, 0, 1.0, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_keep_the_lowest_index(dtype):
    flat = torch.zeros(5, 700, device="cuda", dtype=dtype)
    flat[:, ::2] = -0.0                                               # equal to +0
    u = torch.tensor([0.0, 0.3, 0.5, 0.9, 1 - 2.0 ** -24], device="cuda")
    _check(flat, u, 1.0, 3, 1.0, 0.0)
    _check(flat, u, 1.0, 0, 0.5, 0.0)
    _check(flat, u, 1.0, 699, 0.999, 1.0)
    _check(flat, u, 0.0, 0, 1.0, 0.0)
    steps = flat + (torch.arange(700, device="cuda") % 7 == 3).to(dtype)       # two levels, ties across warps
    _check(steps, u, 1.0, 60, 1.0, 0.0)
    _check(steps, u, 1.0, 150, 0.97, 0.0)
    token, _ = sample(flat, u, 1.0, 3)
    assert token.tolist() == [0, 0, 1, 2, 2]


def test_masked_rows_infinities_and_nan():
    inf = float("inf")
    rows = torch.full((7, 300), -inf, device="cuda")
    rows[1, 250] = -3.0                                               # one token left
    rows[2] = float("nan")
    rows[3, 10], rows[3, 200] = inf, inf                              # all the mass on two
    rows[4, :5] = torch.tensor([1.0, float("nan"), 2.0, -inf, 0.5])
    rows[5] = torch.finfo(torch.float32).min                          # masks of the type's lowest value
    rows[5, 77] = 0.0
    rows[6] = torch.finfo(torch.float32).min
    u = torch.full((7,), 0.6, device="cuda")
    for T, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (inf, 0, 1.0, 0.0),
                       (1e-30, 20, 0.5, 0.1)]:
        if T != inf:
            _check(rows, u, T, k, p, m)
        token, logprob = sample(rows, u, T, k, p, m)
        assert token[0].item() == -1 and token[2].item() == -1 and logprob[0].item() == -inf
        assert token[1].item() == 250 and token[3].item() in (10, 200) and token[5].item() in ((77,) if T != inf else
                                                                                              range(300))
    for dtype in (torch.float16, torch.bfloat16):
        low = torch.full((2, 500), torch.finfo(dtype).min, device="cuda", dtype=dtype)
        low[0, 499] = 1.0
        _check(low, u[:2], 1.0, 0, 0.9, 0.0)


def test_edges_of_the_parameters_and_numbers():
    logits, _ = _logits(4, 513, torch.float32, seed=9)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 2.0 ** -24], device="cuda")
    for T, k, p, m in [(1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 10 ** 9, 1.0, 0.0),
                       (1.0, 513, 1.0, 0.0), (1.0, 512, 1.0, 0.0), (1e-6, 0, 1.0, 0.0), (1e6, 0, 0.3, 0.5),
                       (1.0, 0, 2.0 ** -24, 0.0), (-1.0, 0, 1.0, 0.0)]:
        _check(logits, u, T, k, p, m)


def test_row_strides_and_offsets():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(3, 4, 1001, generator=g).bfloat16().cuda()
    u = torch.rand(3, generator=g).cuda()
    _check(wide[:, -1], u, 0.8, 30, 0.9, 0.0)                         # the last position's logits
    _check(wide[:, 1, 1:], u, 0.8, 30, 0.9, 0.0)                      # rows off every vector boundary
    _check(wide[:, 0, ::2], u, 0.8, 30, 0.9, 0.0)


def test_a_row_does_not_depend_on_its_batch():
    logits, u = _logits(64, 5000, torch.bfloat16, seed=12)
    token, logprob = sample(logits, u, 0.9, 0, 0.95)
    for i in (0, 17, 63):
        t, lp = sample(logits[i:i + 1], u[i:i + 1], 0.9, 0, 0.95)
        assert t.item() == token[i].item() and lp.item() == logprob[i].item()


def test_frequencies_follow_the_probabilities():
    """2^14 evenly spaced numbers draw each token floor/ceil(2^14 p) times."""
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda").expand(1 << 14, 5)
    u = torch.arange(1 << 14, device="cuda").float() / (1 << 14)
    token, _ = sample(logits, u)
    want = torch.softmax(logits[0].double(), 0) * (1 << 14)
    got = torch.bincount(token, minlength=5).double()
    assert float((got - want).abs().max()) <= 1.0


def test_empty_batch_and_refusals():
    t, lp = sample(torch.zeros(0, 10, device="cuda"), torch.zeros(0, device="cuda"))
    assert t.shape == (0,) and lp.shape == (0,)
    l, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        sample(l.cpu(), u.cpu())
    with pytest.raises(RuntimeError, match="u to be float32"):
        sample(l, u[:1])
    with pytest.raises(RuntimeError, match=r"logits \[B,V\]"):
        sample(l[0], u)
    with pytest.raises(RuntimeError, match="top_p"):
        sample(l, u, top_p=torch.zeros(3, device="cuda"))
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        sample(l.double(), u)
    with pytest.raises(RuntimeError, match="unsupported"):
        sample(torch.zeros(1, (1 << 18) + 1, device="cuda"), u[:1])


def test_top_k_beyond_32_bits_keeps_all():
    logits, u = _logits(3, 400, torch.float32, seed=2)
    k = torch.tensor([2 ** 32 + 5, 2 ** 31, -2 ** 33 + 7], device="cuda")
    token, logprob = sample(logits, u, top_k=k)
    want, lp = sample(logits, u)
    assert torch.equal(token, want) and torch.equal(logprob, lp)


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 32000), (torch.float16, 41999), (torch.float32, 20003)])
@pytest.mark.parametrize("T,k,p,m", [(0.8, 50, 0.95, 0.02), (1.0, 400, 0.9, 0.0), (1.0, 0, 0.92, 0.0), (1.7, 4000, 0.99, 0.0),
                                     (1.0, 0, 1.0, 0.0)])
def test_large_vocabularies_of_many_rows(V, T, k, p, m, dtype):
    """Rows enough for a CTA each: a few of them against the definition."""
    logits, u = _logits(80, V, dtype, seed=V + k)
    logits[1, torch.arange(V) % 10 != 3] = float("-inf")
    token, logprob = sample(logits, u, T, k, p, m)
    for i in (0, 1, 79):
        want, lp = _draw(_kept(logits[i], T, k, p, m), u[i].item())
        assert token[i].item() == want and abs(logprob[i].item() - lp) < 1e-5 * max(1.0, abs(lp))


@pytest.mark.parametrize("T,k,p,m", [(0.8, 50, 0.95, 0.02), (1.0, 0, 0.92, 0.0), (1.7, 4000, 0.99, 0.0), (1.0, 0, 1.0, 0.0)])
def test_a_row_is_the_same_in_any_number_of_ctas(T, k, p, m):
    """100 rows have a CTA each, 30 clusters of 2, 12 of 8 and one a cluster of 16."""
    logits, u = _logits(100, 40000, torch.bfloat16, seed=21)
    token, logprob = sample(logits, u, T, k, p, m)
    for n in (30, 12, 1):
        t, lp = sample(logits[:n], u[:n], T, k, p, m)
        assert torch.equal(t, token[:n]) and torch.equal(lp, logprob[:n])
