"""Measured cases of the language-model operators: the gated linear recurrence
(sequence, training step, single token), the gated feed-forward block (prefill,
training step, few tokens) and token sampling.

`run` computes a case through the package's entry points when `own` is true, and by
elementary torch operations in 32 bits (64-bit integers for sampling's masses) when it
is not.  `exact` gives the same results from the definitions in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MASS_ONE = 2 ** 40          # sampling: the mass of the largest logit
FRACTION = 2 ** 24          # sampling: u and top_p are taken in steps of 2^-24


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a training step's recurrence in the LM's width: packed documents (resets), x, gate and output
        # gate as the thirds of one projection
        {"name": "scan train 8x4096x768", "op": "scan_train", "B": 8, "T": 4096, "D": 768, "type": "bf16",
         "packed": True, "resets": True, "lengths": False, "out_gate": True},
        # one long prompt: few channels, so the sequence itself has to be split
        {"name": "scan prefill 1x65536x768", "op": "scan_forward", "B": 1, "T": 65536, "D": 768, "type": "bf16",
         "packed": True, "resets": False, "lengths": False, "out_gate": True},
        # a small right-padded batch in 32 bits, odd sizes, one empty row
        {"name": "scan train ragged f32", "op": "scan_train", "B": 5, "T": 1021, "D": 331, "type": "f32",
         "packed": False, "resets": False, "lengths": True, "out_gate": False},
        # decode: one token for each of the LM's 256 sequences
        {"name": "scan step 256x768", "op": "scan_step", "B": 256, "D": 768, "type": "bf16", "out_gate": True},
        # prefill of the LM's feed-forward: 8 prompts of 2048
        {"name": "ffn prefill 16384x768x768", "op": "ffn_forward", "M": 16384, "D": 768, "F": 768, "type": "bf16",
         "bias": True, "act": "silu"},
        # a training step of a wide block
        {"name": "ffn train 8192x2048x5504", "op": "ffn_train", "M": 8192, "D": 2048, "F": 5504, "type": "bf16",
         "bias": False, "act": "silu"},
        # a training step in the LM's width with an odd number of tokens
        {"name": "ffn train 4099x768x768", "op": "ffn_train", "M": 4099, "D": 768, "F": 768, "type": "bf16",
         "bias": True, "act": "gelu"},
        # decode of one sequence in the LM's width: latency
        {"name": "ffn one token 768x768", "op": "ffn_forward", "M": 1, "D": 768, "F": 768, "type": "bf16",
         "bias": True, "act": "silu"},
        # decode of a small batch in a wide block: the weights' bytes
        {"name": "ffn 13 tokens 2048x5504", "op": "ffn_forward", "M": 13, "D": 2048, "F": 5504, "type": "f16",
         "bias": False, "act": "silu"},
        # decode of the LM: 256 rows of its vocabulary, each with its own parameters
        {"name": "sample 256x32000", "op": "sample", "B": 256, "V": 32000, "type": "bf16", "per_row": True,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02, "masked": 0.0},
        # one sequence, a large vocabulary in 32 bits, nucleus only
        {"name": "sample 1x131072", "op": "sample", "B": 1, "V": 131072, "type": "f32", "per_row": False,
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "masked": 0.0},
        # constrained decoding: most of the vocabulary masked, an odd size, a flat distribution
        {"name": "sample 33x50001 masked", "op": "sample", "B": 33, "V": 50001, "type": "f16", "per_row": False,
         "temperature": 1.7, "top_k": 4000, "top_p": 0.99, "min_p": 0.0, "masked": 0.7},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _not_3072(n, step=1):
    return n + step if n == 3072 else n


def draw(rng):
    op = rng.choice(["scan_train", "scan_forward", "scan_step", "ffn_forward", "ffn_train", "ffn_few", "sample"])
    if op in ("scan_train", "scan_forward"):
        most = 2 ** 26 if op == "scan_forward" else 2 ** 25      # B * T * D
        D = _log_int(rng, 64, 4096)
        if rng.random() < 0.7:
            D = -(-D // 8) * 8
        D = _not_3072(D, 8)
        T = _not_3072(_log_int(rng, 2, min(65536, most // D)))
        B = _log_int(rng, 1, max(1, min(64, most // (D * T))))
        return {"op": op, "B": B, "T": T, "D": D, "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "packed": rng.random() < 0.5, "resets": rng.random() < 0.4, "lengths": rng.random() < 0.3,
                "out_gate": rng.random() < 0.6}
    if op == "scan_step":
        return {"op": op, "B": _log_int(rng, 1, 512), "D": _not_3072(_log_int(rng, 64, 4096)),
                "type": rng.choice(["bf16", "f16", "f32"]), "out_gate": rng.random() < 0.6}
    if op in ("ffn_forward", "ffn_train", "ffn_few"):
        D = _not_3072(8 * _log_int(rng, 16, 512), 8)
        F = _not_3072(8 * _log_int(rng, 16, 1376), 8)
        F = F + 8 if 2 * F == 3072 else F
        if op == "ffn_few":
            M = _log_int(rng, 1, 64)
        else:
            M = _not_3072(_log_int(rng, 64, max(64, min(16384, 9 * 10 ** 10 // (D * F)))))
        return {"op": "ffn_forward" if op == "ffn_few" else op, "M": M, "D": D, "F": F,
                "type": rng.choice(["bf16", "f16"]), "bias": rng.random() < 0.5, "act": rng.choice(["silu", "gelu"])}
    V = _not_3072(_log_int(rng, 1000, 200000))
    return {"op": "sample", "B": _log_int(rng, 1, max(1, min(256, 2 ** 24 // V))), "V": V,
            "type": rng.choice(["bf16", "f16", "f32"]), "per_row": rng.random() < 0.5,
            "temperature": round(rng.uniform(0.5, 1.5), 2), "top_k": rng.choice([0, 20, 50, 500]),
            "top_p": rng.choice([1.0, 0.95, 0.8]), "min_p": rng.choice([0.0, 0.0, 0.05]),
            "masked": rng.choice([0.0, 0.0, 0.9])}


def work(case):
    op = case["op"]
    e = 4 if case["type"] == "f32" else 2
    if op == "scan_step":
        n = case["B"] * case["D"]
        return {"bytes": n * ((4 if case["out_gate"] else 3) * e + 8), "flops": 12 * n}
    if op.startswith("scan"):
        n = case["B"] * case["T"] * case["D"]
        ends = 8 * case["B"] * case["D"]
        og = case["out_gate"]
        if op == "scan_forward":
            return {"bytes": n * (4 if og else 3) * e + ends, "flops": 12 * n}
        # the forward's inputs and output, then dy and one gradient for each input
        return {"bytes": n * ((4 if og else 3) + (4 if og else 3)) * e + 2 * ends, "flops": 40 * n}
    if op.startswith("ffn"):
        M, D, F = case["M"], case["D"], case["F"]
        b = 2 * F if case["bias"] else 0
        if op == "ffn_forward":
            return {"bytes": e * (M * D + 2 * F * D + M * F + b), "flops": 4 * M * D * F}
        return {"bytes": e * (2 * M * D + 4 * F * D + 2 * M * F + 2 * b), "flops": 12 * M * D * F}
    return {"bytes": case["B"] * (case["V"] * e + 4 + 12), "flops": 8 * case["B"] * case["V"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    ty = TYPES[case["type"]]
    op = case["op"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device=DEVICE) * scale + shift

    s = {"case": case}
    if op == "scan_step":
        B, D = case["B"], case["D"]
        k = 3 if case["out_gate"] else 2
        p = normal(B, k, D)
        p[:, 1] = p[:, 1] * 2.0 + 2.0
        p = p.to(ty).view(B, k * D)                     # thirds (or halves) of one projection
        s["x"], s["gate"] = p[:, :D], p[:, D:2 * D]
        s["out_gate"] = p[:, 2 * D:] if case["out_gate"] else None
        s["h"] = normal(B, D)
    elif op.startswith("scan"):
        B, T, D = case["B"], case["T"], case["D"]
        k = 3 if case["out_gate"] else 2
        train = op == "scan_train"
        parts = [normal(B, T, D).to(ty), normal(B, T, D, scale=2.0, shift=2.0).to(ty)]   # gates: memories of 1 to 10^3 steps
        if case["out_gate"]:
            parts.append(normal(B, T, D).to(ty))
        if case["packed"]:
            s["packed"] = torch.cat(parts, dim=-1)
            parts = list(s["packed"].split(D, dim=-1))
            s["packed"].requires_grad_(train)
        s["parts"] = [t.detach().requires_grad_(train and not case["packed"]) for t in parts]
        s["h0"] = normal(B, D).requires_grad_(train)
        s["lengths"] = s["resets"] = None
        if case["lengths"]:
            n = torch.randint(0, T + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
            n[0] = T
            n[B // 2] = 0 if B > 2 else n[B // 2]
            s["lengths"] = n
        if case["resets"]:
            s["resets"] = torch.rand(B, T, generator=g, device=DEVICE) < 1.0 / 512
        if train:
            s["dy"] = normal(B, T, D).to(ty)
            s["dh"] = normal(B, D, scale=0.1)
    elif op.startswith("ffn"):
        M, D, F = case["M"], case["D"], case["F"]
        train = op == "ffn_train"
        s["x"] = normal(M, D).to(ty).requires_grad_(train)
        s["w"] = normal(2 * F, D, scale=1.0 / math.sqrt(D)).to(ty).requires_grad_(train)
        s["b"] = normal(2 * F, scale=0.1).to(ty).requires_grad_(train) if case["bias"] else None
        if train:
            s["dh"] = normal(M, F).to(ty)
    else:
        B, V = case["B"], case["V"]
        logits = normal(B, V, scale=2.5)
        if case["masked"] > 0.0:
            off = torch.rand(B, V, generator=g, device=DEVICE) < case["masked"]
            logits = logits.masked_fill(off, float("-inf"))
        s["logits"] = logits.to(ty)
        s["u"] = torch.randint(0, FRACTION, (B,), generator=g, device=DEVICE).float() / FRACTION
        if case["per_row"]:
            r = torch.rand(4, B, generator=g, device=DEVICE)
            s["temperature"] = case["temperature"] * (0.5 + r[0])
            s["top_k"] = (case["top_k"] * (0.5 + r[1])).to(torch.int32)
            s["top_p"] = (case["top_p"] * (0.8 + 0.2 * r[2])).clamp(max=1.0)
            s["min_p"] = case["min_p"] * r[3]
        else:
            for n in ("temperature", "top_k", "top_p", "min_p"):
                s[n] = case[n]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "scan_step":
        return _step_own(state) if own else _step_plain(state)
    if op.startswith("scan"):
        return _scan_own(state) if own else _scan_plain(state)
    if op.startswith("ffn"):
        return _ffn_own(state) if own else _ffn_plain(state)
    return _sample_own(state) if own else _sample_plain(state)


def _scan_own(s):
    from deltagrid_b200.recurrence import gated_scan, gated_scan_packed
    c = s["case"]
    if c["packed"]:
        y, h = gated_scan_packed(s["packed"], h0=s["h0"], lengths=s["lengths"], resets=s["resets"],
                                 out_gate=c["out_gate"])
        leaves = [s["packed"], s["h0"]]
    else:
        x, gate = s["parts"][:2]
        y, h = gated_scan(x, gate, s["parts"][2] if c["out_gate"] else None, h0=s["h0"], lengths=s["lengths"],
                          resets=s["resets"])
        leaves = [*s["parts"], s["h0"]]
    if c["op"] == "scan_forward":
        return [y, h]
    return [y, h, *torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"]))]


def _step_own(s):
    from deltagrid_b200.recurrence import gated_scan_step
    return [gated_scan_step(s["x"], s["gate"], s["h"], out_gate=s["out_gate"]), s["h"]]


def _ffn_own(s):
    from deltagrid_b200.ffn import gated_ffn
    h = gated_ffn(s["x"], s["w"], s["b"], activation=s["case"]["act"])
    if s["case"]["op"] == "ffn_forward":
        return [h]
    leaves = [s["x"], s["w"]] + ([s["b"]] if s["b"] is not None else [])
    return [h, *torch.autograd.grad(h, leaves, s["dh"])]


def _sample_own(s):
    from deltagrid_b200.sampling import sample
    token, logprob = sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                            min_p=s["min_p"])
    return [token, logprob]


# ---------------------------------------------------------------------------
# plain forms (32 bits)
# ---------------------------------------------------------------------------

def _prefix(c, v):
    """h_t = c_t h_{t-1} + v_t along dim 1, by doubling."""
    d, T = 1, c.shape[1]
    while d < T:
        v = torch.cat([v[:, :d], v[:, d:] + c[:, d:] * v[:, :-d]], 1)
        c = torch.cat([c[:, :d], c[:, d:] * c[:, :-d]], 1)
        d *= 2
    return v


@torch.no_grad()
def _scan_plain(s):
    case = s["case"]
    x, g = s["parts"][0].float(), s["parts"][1].float()
    ty = s["parts"][0].dtype
    T = x.shape[1]
    a = torch.sigmoid(g)
    na = torch.sigmoid(-g)                                  # 1 - a
    keep = torch.ones(x.shape[0], T, 1, device=x.device) if s["resets"] is None else (~s["resets"]).float()[..., None]
    valid = torch.ones(x.shape[0], T, 1, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        valid = (torch.arange(T, device=x.device)[None] < s["lengths"][:, None])[..., None]
    c = torch.where(valid, a * keep, 1.0)
    v = torch.where(valid, na * x, 0.0)
    v[:, 0] += c[:, 0] * s["h0"]
    h = _prefix(c, v)
    h_last = h[:, -1].clone()
    if case["out_gate"]:
        o = s["parts"][2].float()
        so = torch.sigmoid(o)
        y = torch.where(valid, h * o * so, 0.0)
    else:
        y = torch.where(valid, h, 0.0)
    if case["op"] == "scan_forward":
        return [y.to(ty), h_last]
    dy = torch.where(valid, s["dy"].float(), 0.0)
    dh = dy * (o * so) if case["out_gate"] else dy.clone()
    dh[:, -1] += s["dh"]
    cn = torch.cat([c[:, 1:], torch.zeros_like(c[:, :1])], 1)
    d = _prefix(cn.flip(1), dh.flip(1)).flip(1)             # d_t = dh_t + c_{t+1} d_{t+1}
    before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    grads = [torch.where(valid, d * na, 0.0), torch.where(valid, d * (keep * before - x) * a * na, 0.0)]
    if case["out_gate"]:
        grads.append(dy * h * so * (1.0 + o * (1.0 - so)))
    grads = [t.to(ty) for t in grads]
    if case["packed"]:
        grads = [torch.cat(grads, dim=-1)]
    return [y.to(ty), h_last, *grads, c[:, 0] * d[:, 0]]


def _step_plain(s):
    x, g = s["x"].float(), s["gate"].float()
    s["h"].copy_(torch.sigmoid(g) * s["h"] + torch.sigmoid(-g) * x)
    y = s["h"]
    if s["out_gate"] is not None:
        o = s["out_gate"].float()
        y = y * o * torch.sigmoid(o)
    return [y.to(s["x"].dtype), s["h"]]


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        sg = torch.sigmoid(g)
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    k = math.sqrt(2.0 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * g * g)


@torch.no_grad()
def _ffn_plain(s):
    case, ty = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    F = w.shape[0] // 2
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    g, u = z[:, :F], z[:, F:]
    f, df = _act(g, case["act"])
    h = (f * u).to(ty)
    if case["op"] == "ffn_forward":
        return [h]
    dh = s["dh"].float()
    dz = torch.cat([dh * u * df, dh * f], 1)
    out = [h, (dz @ w).to(ty), (dz.t() @ x).to(ty)]
    if s["b"] is not None:
        out.append(dz.sum(0).to(ty))
    return out


def _column(v, like, dtype):
    """A parameter as a [B, 1] column."""
    t = v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((like.shape[0],), v, dtype=dtype, device=like.device)
    return t[:, None]


def _fraction_of(f, n, up):
    """floor (or ceiling) of n * f / 2^24 for whole f <= 2^24 and n < 2^58."""
    low = f * (n % FRACTION) + (FRACTION - 1 if up else 0)
    return f * (n // FRACTION) + low // FRACTION


def _sample_plain(s):
    l = s["logits"].float()
    B, V = l.shape
    l = torch.where(torch.isnan(l), float("-inf"), l)
    temperature = _column(s["temperature"], l, torch.float32)
    m = l.max(dim=1, keepdim=True).values
    z = torch.where(l == m, 0.0, (l - m) / torch.where(temperature > 0, temperature, 1.0))
    w = (torch.exp(z) * MASS_ONE).to(torch.int64)
    w = torch.where(torch.isneginf(l), 0, w)
    greedy = temperature <= 0
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    sorted_w = torch.gather(w, 1, order)
    k = _column(s["top_k"], l, torch.int64)
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > V), V, k))
    keep = torch.arange(V, device=l.device)[None] < k
    run_w = torch.cumsum(torch.where(keep, sorted_w, 0), 1)
    p = (_column(s["top_p"], l, torch.float32).clamp(0.0, 1.0) * FRACTION).to(torch.int64)
    keep &= run_w - sorted_w < _fraction_of(p, run_w[:, -1:], True).clamp(min=1)
    least = (_column(s["min_p"], l, torch.float32).clamp(0.0, 1.0) * MASS_ONE).to(torch.int64)
    keep &= sorted_w >= least
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0)
    run_w = torch.cumsum(w, 1)
    total = run_w[:, -1:]
    at = _fraction_of((s["u"].clamp(0.0, 1.0 - 1.0 / FRACTION) * FRACTION).to(torch.int64)[:, None], total, False)
    token = (run_w <= at).sum(1)
    none = total[:, 0] == 0
    mass = torch.gather(w, 1, token.clamp(max=V - 1)[:, None])[:, 0].float()
    logprob = torch.where(none, float("-inf"), torch.log(mass / total[:, 0].float()))
    return [torch.where(none, -1, token), logprob]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "scan_step":
        a = 1.0 / (1.0 + torch.exp(-s["gate"].double()))
        h = a * s["h"].double() + (1.0 - a) * s["x"].double()
        return [h if s["out_gate"] is None else h * _swish64(s["out_gate"].double()), h]
    if case["op"].startswith("scan"):
        return _scan_exact(s)
    if case["op"].startswith("ffn"):
        return _ffn_exact(s)
    return [None, _logprob_exact(s)]


def _swish64(o):
    return o / (1.0 + torch.exp(-o))


def _scan_exact(s):
    """One step after another, then back."""
    case = s["case"]
    x = s["parts"][0].double()
    a = 1.0 / (1.0 + torch.exp(-s["parts"][1].double()))
    B, T, D = x.shape
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=x.device)
    live = torch.arange(T, device=x.device)[None] < n[:, None]
    carry = a if s["resets"] is None else a * (~s["resets"])[..., None]
    h = s["h0"].double()
    before, after = torch.empty_like(x), torch.empty_like(x)
    ragged = s["lengths"] is not None
    add = (1.0 - a) * x
    for t in range(T):
        before[:, t] = h
        new = torch.addcmul(add[:, t], carry[:, t], h)
        h = torch.where(live[:, t, None], new, h) if ragged else new
        after[:, t] = h
    gate = _swish64(s["parts"][2].double()) if case["out_gate"] else torch.ones_like(x)
    y = after * gate * live[..., None]
    if case["op"] == "scan_forward":
        return [y, h]
    dy = s["dy"].double() * live[..., None]
    din = dy * gate
    d = s["dh"].double().clone()
    total = torch.zeros_like(x)
    for t in reversed(range(T)):
        here = d + din[:, t]
        total[:, t] = here
        back = here * carry[:, t]
        d = torch.where(live[:, t, None], back, d) if ragged else back
    total = total * live[..., None]
    grads = [total * (1.0 - a), total * (carry / a * before - x) * a * (1.0 - a)]
    if case["out_gate"]:
        o = s["parts"][2].double()
        e = 1.0 / (1.0 + torch.exp(-o))
        grads.append(dy * after * (e + o * e * (1.0 - e)))
    if case["packed"]:
        grads = [torch.cat(grads, dim=-1)]
    return [y, h, *grads, d]


def _ffn_exact(s):
    case = s["case"]
    x, w = s["x"].double(), s["w"].double()
    wg, wu = w.chunk(2, dim=0)
    g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    if s["b"] is not None:
        bg, bu = s["b"].double().chunk(2)
        g += bg
        u += bu
    if case["act"] == "silu":
        e = 1.0 / (1.0 + torch.exp(-g))
        f = g * e
        slope = e + f * (1.0 - e)
    else:
        k = math.sqrt(2.0 / math.pi)
        e = torch.tanh(k * (g + 0.044715 * g ** 3))
        f = g * (1.0 + e) / 2
        slope = (1.0 + e) / 2 + g / 2 * (1.0 - e ** 2) * k * (1.0 + 0.134145 * g ** 2)
    if case["op"] == "ffn_forward":
        return [f * u]
    dh = s["dh"].double()
    dg, du = dh * u * slope, dh * f
    out = [f * u, torch.mm(dg, wg) + torch.mm(du, wu), torch.cat([torch.mm(dg.t(), x), torch.mm(du.t(), x)])]
    if s["b"] is not None:
        out.append(torch.cat([dg.sum(0), du.sum(0)]))
    return out


def _logprob_exact(s):
    """The log-probability of the drawn token, row by row with 64-bit masses."""
    rows = []
    B, V = s["logits"].shape

    def of(name, i):
        v = s[name]
        return float(v[i]) if isinstance(v, torch.Tensor) else float(v)

    for i in range(B):
        l = s["logits"][i].double()
        T = of("temperature", i)
        w = torch.exp((l - l.max()) / T)
        w = torch.where(w * MASS_ONE < 1.0, 0.0, w)
        value, order = torch.sort(l, descending=True, stable=True)
        k = int(of("top_k", i))
        k = k if 0 < k < V else V
        ws = w[order[:k]]
        p = math.floor(of("top_p", i) * FRACTION) / FRACTION
        ws = torch.where(torch.cumsum(ws, 0) - ws < max(p * float(ws.sum()), 1.0 / MASS_ONE), ws, 0.0)
        ws = torch.where(ws >= of("min_p", i), ws, 0.0)
        kept = torch.zeros_like(w)
        kept[order[:k]] = ws
        c = torch.cumsum(kept, 0)
        token = int((c <= float(s["u"][i]) * float(c[-1])).sum())
        rows.append(torch.log(kept[min(token, V - 1)] / c[-1]))
    return torch.stack(rows)
