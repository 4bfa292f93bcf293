"""HybridLM: the gated recurrence, the memory layer, the feed-forward block and sampling run
together.  Sequence and token-by-token forms agree within 2e-3 (32-bit arithmetic in two
orders through four blocks; the memory layer's own forward / step bar is 1e-4 in 32 bits)."""
import pytest
import torch
import torch.nn.functional as F

from conftest import rel_err

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from deltagrid_b200.hybrid import HybridLM
    from deltagrid_b200.sampling import sample


def _model(dtype=torch.float32, **kw):
    torch.manual_seed(0)
    return HybridLM(97, d_model=64, layers=4, num_heads=2, **kw).cuda().to(dtype)


def test_step_continues_forward():
    m = _model().eval()
    ids = torch.randint(0, 97, (3, 12), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        full, _ = m(ids)
        logits, states = m(ids[:, :5])
        outs = [logits[:, -1]]
        for t in range(5, 12):
            logits, states = m.step(ids[:, t], states)
            outs.append(logits)
    assert rel_err(torch.stack(outs, 1).cpu(), full[:, 4:].cpu()) < 2e-3


def test_a_step_of_training_lowers_the_loss():
    m = _model()
    ids = torch.randint(0, 97, (4, 40), generator=torch.Generator().manual_seed(2)).cuda()
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    losses = []
    for _ in range(4):
        logits, _ = m(ids[:, :-1])
        loss = F.cross_entropy(logits.reshape(-1, 97), ids[:, 1:].reshape(-1))
        opt.zero_grad(set_to_none=True)
        loss.backward()
        used = [p for n, p in m.named_parameters() if p.requires_grad and "decay" not in n]
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in used)
        opt.step()
        losses.append(loss.item())
    assert losses == sorted(losses, reverse=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_generate_is_the_loop_and_repeats(dtype):
    m = _model(dtype).eval()
    ids = torch.randint(0, 97, (2, 6), generator=torch.Generator().manual_seed(3)).cuda()
    u = torch.rand(2, 5, generator=torch.Generator().manual_seed(4)).cuda()
    args = dict(temperature=0.9, top_k=20, top_p=0.9, min_p=0.01)
    tokens, logprobs = m.generate(ids, 5, u=u, **args)
    with torch.no_grad():
        logits, states = m(ids)
        logits = logits[:, -1]
        for i in range(5):
            t, lp = sample(logits, u[:, i], 0.9, 20, 0.9, 0.01)
            assert torch.equal(t, tokens[:, i]) and torch.equal(lp, logprobs[:, i])
            logits, states = m.step(t, states)
    again, _ = m.generate(ids, 5, u=u, **args)
    assert torch.equal(tokens, again)
    a, _ = m.generate(ids, 4, generator=torch.Generator(device="cuda").manual_seed(7))
    b, _ = m.generate(ids, 4, generator=torch.Generator(device="cuda").manual_seed(7))
    assert torch.equal(a, b)


def test_refusals():
    m = _model()
    with pytest.raises(ValueError, match="prompts"):
        m.generate(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), 3)
    with pytest.raises(ValueError, match="expected u"):
        m.generate(torch.zeros(2, 1, dtype=torch.int64, device="cuda"), 3, u=torch.zeros(2, 2, device="cuda"))
    with pytest.raises(ValueError, match="kind"):
        from deltagrid_b200.hybrid import HybridBlock
        HybridBlock("attention", 64, 2, None, None)
    t, lp = m.generate(torch.zeros(2, 1, dtype=torch.int64, device="cuda"), 0)
    assert t.shape == (2, 0) and lp.shape == (2, 0)


def test_generate_where_nothing_can_be_drawn():
    m = _model().eval()
    ids = torch.randint(0, 97, (3, 4), generator=torch.Generator().manual_seed(5)).cuda()
    with torch.no_grad():
        m.head.weight.fill_(float("nan"))
    tokens, logprobs = m.generate(ids, 3)
    torch.cuda.synchronize()
    assert (tokens == -1).all() and torch.isneginf(logprobs).all()


def test_resets_are_refused_by_delta_blocks():
    """The memory layer has no resets: its state would flow from document to document."""
    from deltagrid_b200.hybrid import HybridBlock
    x = torch.zeros(2, 5, 64, device="cuda")
    r = torch.zeros(2, 5, dtype=torch.bool, device="cuda")
    HybridBlock("recurrence", 64, 2, None, None).cuda()(x, resets=r)
    b = HybridBlock("delta", 64, 2, None, None).cuda()
    b(x)
    with pytest.raises(ValueError, match="resets"):
        b(x, resets=r)
