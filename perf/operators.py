"""The operators on 4-bit weights (ultraquant_b200.q4): what is measured of them, and their plain forms.

A weight matrix (N, K) is held as w[n, k] = s * e[n, k // g] * q[n, k]: q whole numbers in -8 .. 7, e one E4M3 value for
each group of g along a row, s one float32 for the matrix.  Eight codes u = q + 8 fill four bytes; the low halves of the
bytes hold elements 0, 4, 1, 5 and the high halves 2, 6, 3, 7.

Kinds of case: "linear" (y = x W^T, with its backward pass where "train"), "experts" (the same product for the rows of
each expert, ragged), "embedding" (rows by token, scaled, with the gradient of the group scales where "train") and
"codec" (weights to codes and back)."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a square projection (attention output of a 4096-wide model): latency counts
        {"name": "linear 1 token", "kind": "linear", "T": 1, "N": 4096, "K": 4096, "group": 32, "dtype": "bf16", "train": False},
        # a small batch of sequences, one token each, through an odd-sized up projection
        {"name": "linear 7 tokens, odd sizes", "kind": "linear", "T": 7, "N": 14331, "K": 4128, "group": 32, "dtype": "fp16", "train": False},
        # a prompt through the up projection of an 8B-sized model
        {"name": "linear prompt", "kind": "linear", "T": 2047, "N": 14336, "K": 4096, "group": 128, "dtype": "bf16", "train": False},
        # tuning the group scales of the down projection, codes fixed: forward and both gradients
        {"name": "linear tuning step", "kind": "linear", "T": 4096, "N": 4096, "K": 14336, "group": 32, "dtype": "bf16", "train": True},
        # a decode batch over many small experts, some without a row
        {"name": "experts decode", "kind": "experts", "E": 64, "active": 51, "T": 96, "N": 2048, "K": 4096, "group": 32, "dtype": "bf16", "train": False},
        # a prompt over large experts, uneven loads
        {"name": "experts prompt", "kind": "experts", "E": 16, "active": 15, "T": 8191, "N": 4096, "K": 4096, "group": 256, "dtype": "bf16", "train": False},
        # tuning the experts' group scales
        {"name": "experts tuning step", "kind": "experts", "E": 8, "active": 8, "T": 6001, "N": 4096, "K": 2048, "group": 64, "dtype": "fp16", "train": True},
        # the next tokens of three sequences
        {"name": "embedding 3 tokens", "kind": "embedding", "T": 3, "V": 32000, "K": 4096, "group": 32, "dtype": "bf16", "train": False},
        # a batch of prompts
        {"name": "embedding prompts", "kind": "embedding", "T": 16384, "V": 65537, "K": 4096, "group": 64, "dtype": "fp16", "train": False},
        # a tuning batch: lookup and the gradient of the table's group scales; tokens as frequent as words are
        {"name": "embedding tuning step", "kind": "embedding", "T": 16384, "V": 131072, "K": 4096, "group": 32, "dtype": "bf16", "train": True},
        # quantizing a small projection stored in 16 bits
        {"name": "codec small", "kind": "codec", "N": 1024, "K": 4096, "group": 256, "dtype": "bf16"},
        # quantizing the down projection of an 8B-sized model
        {"name": "codec large", "kind": "codec", "N": 4096, "K": 14336, "group": 32, "dtype": "fp32"},
    ]


def _between(rng, lo, hi):
    """A whole number, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "embedding", "codec"])
    group = rng.choice([32, 64, 128, 256])
    K = max(1, round(_between(rng, 256, 14336) / group)) * group
    case = {"kind": kind, "group": group, "dtype": rng.choice(["bf16", "fp16"])}
    if kind == "embedding":
        return dict(case, T=_between(rng, 1, 16384), V=_between(rng, 1000, 131072), K=min(K, 4096), train=rng.random() < 0.5)
    if kind == "codec":
        return dict(case, N=_between(rng, 100, 4096), K=K, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    train = rng.random() < 0.4
    if kind == "linear":
        N = _between(rng, 257, 14336)
        most = max(1, min(8192, int((2.4e11 if train else 7e11) / (N * K))))
        return dict(case, T=_between(rng, 1, most), N=N, K=K, train=train)
    E = _between(rng, 2, 64)
    N = _between(rng, 257, 4096)
    K = min(K, max(1, int(6e8 / (E * N)) // group) * group)
    most = max(E, min(8192, int(1.4e11 / (N * K))))
    return dict(case, E=E, active=rng.randint(max(1, E // 2), E), T=_between(rng, E, most), N=N, K=K, train=train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    kind = case["kind"]
    K, group = case["K"], case["group"]
    if kind == "codec":
        # Gaussian weights with rows of different size and a few outliers
        w = torch.randn(case["N"], K, generator=g, device="cuda") * 0.02
        w *= torch.exp(0.5 * torch.randn(case["N"], 1, generator=g, device="cuda"))
        w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 1e-3, 8 * w, w)
        return {"case": case, "w": w.to(dt)}
    rows = case["V"] if kind == "embedding" else case["N"]
    E = case.get("E", 1)
    # codes as the encoder leaves them: Gaussian weights over a group scale of a third of the largest
    codes = torch.empty(E * rows, K // 2, dtype=torch.uint8, device="cuda")
    for at in range(0, E * rows, 16384):
        part = codes[at : at + 16384]
        q = torch.randn(2, *part.shape, generator=g, device="cuda").mul_(2.9).round_().clamp_(-8, 7).to(torch.int8) + 8
        part.copy_((q[0] | q[1] << 4).to(torch.uint8))
    e = torch.exp(0.3 * torch.randn(E * rows, K // group, generator=g, device="cuda")) * 40
    e *= 1 - 2 * torch.randint(0, 2, e.shape, generator=g, device="cuda")
    state = {"case": case, "codes": codes.view(E, rows, K // 2), "e": e.to(torch.float8_e4m3fn).view(E, rows, K // group)}
    state["s"] = torch.full((E,), 2.0**-12, device="cuda") * torch.exp2(torch.randint(-1, 2, (E,), generator=g, device="cuda").float())
    T = case["T"]
    if kind == "embedding":
        state = {k: v[0] if k in ("codes", "e", "s") else v for k, v in state.items()}
        # token v as frequent as 1 / (v + 3): words by rank, the ranks spread over the table
        u = torch.rand(T, generator=g, device="cuda", dtype=torch.float64)
        rank = (3 * torch.exp(u * math.log((case["V"] + 3) / 3)) - 3).long().clamp_(0, case["V"] - 1)
        state["tokens"] = torch.randperm(case["V"], generator=g, device="cuda")[rank]
        if case["train"]:
            state["dy"] = (torch.randn(T, K, generator=g, device="cuda") * 0.1).to(dt)
    else:
        # activations behind a norm: unit size, a few channels larger
        x = torch.randn(T, K, generator=g, device="cuda") * (1 + 4 * (torch.rand(K, generator=g, device="cuda") < 0.01))
        state["x"] = x.to(dt)
        if case["train"]:
            state["dy"] = (torch.randn(T, case["N"], generator=g, device="cuda") * 0.1).to(dt)
    if kind == "experts":
        # every active expert has a row; the others are shared out unevenly
        A = case["active"]
        on = torch.randperm(E, generator=g, device="cuda")[:A]
        size = torch.exp(0.7 * torch.randn(A, generator=g, device="cuda"))
        more = torch.multinomial(size, T - A, replacement=True, generator=g) if T > A else on[:0]
        count = torch.zeros(E, dtype=torch.long, device="cuda")
        count[on] = 1 + torch.bincount(more, minlength=A)
        state["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
        state["most"] = int(count.max())
    elif kind == "linear":
        state = {k: v[0] if k in ("codes", "e", "s") else v for k, v in state.items()}
    if case["train"]:
        # the group scales that are trained: float32, of which e holds the rounding
        state["scales"] = state["e"].float() * state["s"][..., None, None]
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _q(codes):
    """(..., K/2) bytes -> (..., K) float32 whole numbers."""
    b = codes.unflatten(-1, (-1, 4))
    lo, hi = (b & 15)[..., [0, 2]], (b >> 4)[..., [0, 2]]  # elements 0, 1 and 2, 3
    lo2, hi2 = (b & 15)[..., [1, 3]], (b >> 4)[..., [1, 3]]  # elements 4, 5 and 6, 7
    return torch.cat([lo, hi, lo2, hi2], -1).flatten(-2).float() - 8


def _w(codes, e, s):
    q = _q(codes)
    c = e.float() * s[..., None, None]
    return (q.unflatten(-1, (c.shape[-1], -1)) * c[..., None]).flatten(-2)


def _plain_linear(st):
    x, dt = st["x"].float(), st["x"].dtype
    w = _w(st["codes"], st["e"], st["s"])
    y = (x @ w.T).to(dt)
    if not st["case"]["train"]:
        return [y]
    dy = st["dy"].float()
    dc = ((dy.T @ x) * _q(st["codes"])).unflatten(-1, (st["e"].shape[-1], -1)).sum(-1)
    return [y, (dy @ w).to(dt), dc]


def _plain_experts(st):
    x, dt, most = st["x"].float(), st["x"].dtype, st["most"]
    off = st["offsets"].long()
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(off, row, right=True) - 1
    at = row - off[expert]
    w = _w(st["codes"], st["e"], st["s"])
    xs = x.new_zeros(w.shape[0], most, x.shape[1])
    xs[expert, at] = x
    y = torch.bmm(xs, w.transpose(1, 2))[expert, at].to(dt)
    if not st["case"]["train"]:
        return [y]
    ds = x.new_zeros(w.shape[0], most, w.shape[1])
    ds[expert, at] = st["dy"].float()
    dc = (torch.bmm(ds.transpose(1, 2), xs) * _q(st["codes"])).unflatten(-1, (st["e"].shape[-1], -1)).sum(-1)
    return [y, torch.bmm(ds, w)[expert, at].to(dt), dc]


ALPHA = 1.5  # the factor on looked-up rows


def _plain_embedding(st):
    c = st["e"].float() * st["s"]
    rows = _q(st["codes"][st["tokens"]]).unflatten(-1, (c.shape[-1], -1))
    y = (rows * (ALPHA * c[st["tokens"]])[..., None]).flatten(-2).to(TYPES[st["case"]["dtype"]])
    if not st["case"]["train"]:
        return [y]
    part = (rows.double() * st["dy"].unflatten(-1, (c.shape[-1], -1)).double()).sum(-1)  # long sums of frequent tokens: 64 bits
    dc = torch.zeros(c.shape, dtype=torch.float64, device=c.device).index_add_(0, st["tokens"], part)
    return [y, (ALPHA * dc).float()]


def _plain_codec(st):
    x = st["w"].float().unflatten(-1, (-1, st["case"]["group"]))
    top = x.abs().amax()
    m, ex = torch.frexp(top)  # top = m 2^ex, m in [1/2, 1): the least power of two s with top <= 3584 s
    s = torch.ldexp(torch.ones_like(top), ex - torch.where(m <= 0.875, 12, 11))
    big = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    e = (-big / (8 * s)).to(torch.float8_e4m3fn).float()
    e = torch.where((e == 0) & (big != 0), torch.copysign(torch.full_like(e, 2.0**-9), -big), e)
    c = (e * s).double()
    q = torch.where(c == 0, 0.0, (x.double() / c).round().clamp(-8, 7))  # in 64 bits: values next to a border
    return [(q * c).float().flatten(-2)]


def _own(st):
    from ultraquant_b200 import q4

    kind = st["case"]["kind"]
    if kind == "codec":
        return [q4.deq_q4(q4.enc_q4(st["w"], st["case"]["group"]))]
    w = q4.Q4(st["codes"], st["e"], st["s"])
    train = st["case"]["train"]
    scales = st["scales"].detach().requires_grad_() if train else None
    if kind == "embedding":
        y = q4.embedding(st["tokens"], w, ALPHA, scales, dtype=TYPES[st["case"]["dtype"]])
        return [y.detach(), *torch.autograd.grad(y, (scales,), st["dy"])] if train else [y]
    x = st["x"].detach().requires_grad_() if train else st["x"]
    y = q4.linear(x, w, scales) if kind == "linear" else q4.grouped_linear(x, st["offsets"], w, scales)
    return [y.detach(), *torch.autograd.grad(y, (x, scales), st["dy"])] if train else [y]


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "experts": _plain_experts, "embedding": _plain_embedding, "codec": _plain_codec}[state["case"]["kind"]](state)


def work(case):
    K, group = case["K"], case["group"]
    wide = 4 if case["dtype"] == "fp32" else 2
    per_row = K / 2 + K / group  # bytes of one row of codes and scales
    if case["kind"] == "codec":
        n = case["N"] * K
        return {"bytes": n * wide + 2 * case["N"] * per_row + 4 * n, "flops": 8 * n}
    T = case["T"]
    if case["kind"] == "embedding":
        b, f = T * (8 + per_row + K * wide), 2 * T * K
        if case["train"]:
            b, f = b + T * (8 + K * wide + K / 2) + 4 * case["V"] * K / group, f + 3 * T * K
        return {"bytes": b, "flops": f}
    N, A, E = case["N"], case.get("active", 1), case.get("E", 1)
    b = A * N * per_row + T * (K + N) * wide
    if case["train"]:
        # the codes again, both gradients of the step's size, and the scales' gradient of every expert
        b += A * N * per_row + T * (K + N) * wide + T * K * wide + 4 * E * N * K / group
    return {"bytes": b, "flops": 2 * T * N * K * (3 if case["train"] else 1)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _exact_q(codes):
    """Whole numbers by a table of what each byte and place of a word holds, float64."""
    b = codes.long()
    out = torch.empty(*b.shape[:-1], b.shape[-1] * 2, dtype=torch.float64, device=b.device)
    for place, (low, high) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        out[..., low::8] = (b[..., place::4] % 16 - 8).double()
        out[..., high::8] = (b[..., place::4] // 16 - 8).double()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    group = case["group"]
    if case["kind"] == "codec":
        w = st["w"].double()
        top = float(w.abs().max())
        s = 2.0 ** math.ceil(math.log2(top / 3584))
        out = torch.empty_like(w)
        grid = torch.tensor([(8 + m) / 8 * 2.0**p for p in range(-6, 9) for m in range(8)][:-1], dtype=torch.float64, device="cuda")
        grid = torch.cat([torch.arange(1, 8, dtype=torch.float64, device="cuda") / 512, grid])  # E4M3, positive
        for j in range(0, case["K"], group):
            x = w[:, j : j + group]
            big = x.gather(1, x.abs().max(1, keepdim=True).indices)
            # the first of the largest: argmax of a tensor of ties gives the lowest place
            big = torch.where(big.abs() > 0, x.gather(1, (x.abs() == big.abs()).long().argmax(1, keepdim=True)), big)
            t = (big.abs() / (8 * s)).flatten()
            up = torch.searchsorted(grid, t).clamp(1, len(grid) - 1)
            lo, hi = grid[up - 1], grid[up]
            even = (up % 2 == 1)  # the grid's places 0, 2, ... are odd in the last bit
            e = torch.where((t - lo > hi - t) | ((t - lo == hi - t) & even), hi, lo)
            c = -torch.sign(big) * s * e[:, None]
            out[:, j : j + group] = torch.where(c == 0, 0.0, torch.round(x / c).clamp(-8, 7) * c)
        return [out]
    if case["kind"] == "embedding":
        tok = st["tokens"]
        q = _exact_q(st["codes"][tok])
        c = st["e"].double() * st["s"].double()
        y = q * c[tok].repeat_interleave(group, 1) * ALPHA
        if not case["train"]:
            return [y]
        order = torch.argsort(tok)
        part = (q * st["dy"].double())[order].view(len(tok), -1, group).sum(2).cumsum(0) * ALPHA
        last = torch.cat([tok[order][1:] != tok[order][:-1], torch.ones(1, dtype=torch.bool, device=tok.device)])
        total = part[last]
        dc = torch.zeros_like(c)
        dc[tok[order][last]] = total - torch.cat([torch.zeros_like(total[:1]), total[:-1]])
        return [y, dc]
    E = case.get("E", 1)
    codes, e, s = (st[k].reshape(E, *st[k].shape[-2:]) if k != "s" else st[k].reshape(E) for k in ("codes", "e", "s"))
    off = st["offsets"].tolist() if "offsets" in st else [0, case["T"]]
    x = st["x"].double()
    y = torch.zeros(case["T"], case["N"], dtype=torch.float64, device="cuda")
    dx, dc = torch.zeros_like(x), torch.zeros(e.shape, dtype=torch.float64, device="cuda")
    for i in range(E):
        a, b = off[i], off[i + 1]
        if a == b:
            continue
        q = _exact_q(codes[i])
        w = q * (e[i].double() * s[i].double()).repeat_interleave(group, 1)
        y[a:b] = x[a:b] @ w.T
        if case["train"]:
            d = st["dy"][a:b].double()
            dx[a:b] = d @ w
            dc[i] = (torch.einsum("tn,tk->nk", d, x[a:b]) * q).view(case["N"], -1, group).sum(2)
    return [y, dx, dc.view(st["e"].shape)] if case["train"] else [y]
