"""The operators of a verify layer that keeps a recurrent state, and of acceptance by the target's probabilities, as cases
that a timer can run: the gated delta rule (decode steps, prefill, and the verify of a tree of drafted tokens with the commit
of its accepted path), the 8-bit integer matrix product with a scale for each token and channel, the norms around a block
with its gate, residual and 8-bit output, and the acceptance of drafted tokens by rejection sampling.

With `own` false `run` computes the plain forms (elementary torch operations in 32 bits; 64 where a border decides a whole
number, and for the inverse of a triangle); with `own` true it makes the framework's calls.

Sizes: hidden 4096 and 2560 (the framework's two layer layouts), heads of 64 and 128. Token counts: 1 (decode), 6 (a verify
of five drafts), up to 24 drafted tokens a sequence (a tree), 8192 (a prompt). Vocabularies of 5000 to 248,320.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One conversation's next token through a layer: the smallest call, latency only.
        step("delta_decode_one", 1, 1, 16, 32, 128),
        # A serving batch's next tokens: the states' bytes both ways.
        step("delta_decode_batch", 48, 1, 16, 32, 128),
        # Prompts of mixed lengths in one call.
        step("delta_prefill_ragged", 5, 700, 8, 16, 128),
        # A long prompt: one sequence, a state at a time from one end to the other.
        step("delta_prefill_long", 1, 8192, 16, 32, 128),
        # One conversation's verify of five drafts and the commit of what was accepted.
        verify("delta_verify_chain", 1, 6, 16, 32, 128, "chain"),
        # A serving batch's trees of up to 24 drafts, and their accepted paths.
        verify("delta_verify_tree", 24, 24, 16, 32, 128, "tree"),
        # A verify's query, key, value and gate projection.
        linear("int8_verify", 6, 12288, 4096, "bf16"),
        # The ragged last chunk of a prompt through it.
        linear("int8_prefill", 1531, 12288, 4096, "bf16"),
        # The norms around a verify's block: of its output, with the residual, and ahead of the next one.
        norm("norm_verify", 6, 4096, "bf16", 0, True, "none", True, True),
        # A prefill chunk's heads: normed one by one, gated, as codes for the output projection.
        norm("norm_prefill", 2048, 4096, "bf16", 128, True, "silu", False, False),
        # One conversation's drafts from a head that proposes its best token: acceptance by the target alone.
        accept("accept_one", 1, 6, 151936, 0, "f32"),
        # A batch of conversations with sampled drafts.
        accept("accept_batch", 16, 6, 151936, 120000, "f32"),
    ]


def step(name, B, L, Hk, Hv, D):
    return {"name": name, "kind": "step", "B": B, "L": L, "Hk": Hk, "Hv": Hv, "D": D}


def verify(name, B, n, Hk, Hv, D, shape):
    return {"name": name, "kind": "verify", "B": B, "L": n, "Hk": Hk, "Hv": Hv, "D": D, "shape": shape}


def linear(name, M, N, K, out):
    return {"name": name, "kind": "linear", "M": M, "N": N, "K": K, "out": out}


def norm(name, M, K, act, group, gate, gate_act, residual, pre):
    """group 0: the first norm is over the whole row."""
    return {"name": name, "kind": "norm", "M": M, "K": K, "act": act, "group": group, "gate": gate, "gate_act": gate_act,
            "residual": residual, "pre": pre}


def accept(name, B, n, V, Vd, act):
    """n: rows of the largest sequence (its drafts and one more). Vd: the draft's vocabulary, 0: no draft probabilities."""
    return {"name": name, "kind": "accept", "B": B, "n": n, "V": V, "Vd": Vd, "act": act}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["step"] * 3 + ["verify"] * 2 + ["linear"] * 2 + ["norm"] * 2 + ["accept"] * 2)
    if kind in ("step", "verify"):
        Hk = rng.choice([1, 2, 4, 8, 16])
        Hv, D = Hk * rng.choice([1, 2, 2, 3, 4] if Hk <= 8 else [1, 2]), rng.choice([64, 128])
        if kind == "verify":
            case = verify("", _log_int(rng, 1, 24), _log_int(rng, 1, 24), Hk, Hv, D, rng.choice(["chain", "tree"]))
        elif rng.random() < 0.5:
            case = step("", _log_int(rng, 1, 48), rng.choice([1, 1, rng.randint(2, 16)]), Hk, Hv, D)
        else:
            B = rng.choice([1, 1, rng.randint(2, 8)])
            case = step("", B, _log_int(rng, 17, 8192 // B), Hk, Hv, D)
    elif kind == "linear":
        N = rng.choice([_log_int(rng, 300, 12288), 16 * _log_int(rng, 20, 700), 256 * rng.randint(2, 48)])
        K = rng.choice([1024, 2048, 2560, 4096, 16 * rng.randint(8, 256)])
        case = linear("", _log_int(rng, 1, 1531), N, K, rng.choice(["bf16", "bf16", "f32"]))
    elif kind == "norm":
        group = rng.choice([0, 0, 64, 128])
        K = rng.choice([2560, 4096, (group or 16) * rng.randint(4, 4096 // (group or 16))])
        case = norm("", _log_int(rng, 1, 2048), K, rng.choice(["bf16", "bf16", "f32"]), group, rng.random() < 0.6,
                    rng.choice(["none", "silu", "sigmoid"]), rng.random() < 0.6, rng.random() < 0.6)
    else:
        V = rng.choice([5000, 151936, 248320, _log_int(rng, 1000, 150000)])
        Vd = rng.choice([0, V, V * 3 // 4])
        n = _log_int(rng, 1, 16)
        case = accept("", _log_int(rng, 1, min(32, max(1, 96 * 271936 // (n * (V + Vd))))), n, V, Vd, rng.choice(["f32", "f32", "bf16"]))
    case.pop("name")
    return case


# ---- inputs ----

def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _randn(shape, g):
    return torch.randn(shape, device="cuda", generator=g)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case):
    """Tokens of each sequence (the first has the most): the same for every seed, so that outputs have one shape."""
    most = case["L"] if "L" in case else case["n"]
    return [most] + torch.randint(1, most + 1, (case["B"] - 1,), generator=_gen(most, "cpu")).tolist()


def _starts(news):
    return _i32([0] + torch.tensor(news).cumsum(0).tolist())


def prepare(case, seed):
    seed = 1000 * seed + 31
    g, host = _gen(seed), _gen(seed + 1, "cpu")
    kind = case["kind"]
    if kind in ("step", "verify"):
        B, Hk, Hv, D = (case[x] for x in ("B", "Hk", "Hv", "D"))
        news = _lengths(case)
        T = sum(news)
        qkv = _randn((T, 2 * Hk + Hv, D), g).to(torch.bfloat16)  # one projection's output: the views are strided
        gates = _randn((T, 2 * Hv), g).to(torch.bfloat16)
        rate = 1.0 + 15.0 * torch.rand(Hv, device="cuda", generator=g)
        dt = torch.exp(torch.rand(Hv, device="cuda", generator=g) * math.log(100.0) + math.log(0.001))
        s = {"case": case, "q": qkv[:, :Hk], "k": qkv[:, Hk:2 * Hk], "v": qkv[:, 2 * Hk:], "a": gates[:, :Hv],
             "b": gates[:, Hv:], "A_log": torch.log(rate), "dt_bias": torch.log(torch.expm1(dt)),
             "state": 0.3 * _randn((B + 2, Hv, D, D), g), "starts": _starts(news),
             "slots": torch.randperm(B + 2, generator=host)[:B].to(torch.int32).cuda()}  # a pool of states, some not in use
        if kind == "verify":
            if case["shape"] == "tree":
                parents = [[-1] + [int(torch.randint(max(-1, i - 6), i, (1,), generator=host)) for i in range(1, c)] for c in news]
            else:
                parents = [list(range(-1, c - 1)) for c in news]
            kept = [_path(p, host) for p in parents]
            path = torch.zeros(B, case["L"], dtype=torch.int32)
            for i, p in enumerate(kept):
                path[i, :len(p)] = torch.tensor(p)
            s.update(mask=_mask(parents), path=path.cuda(), count=_i32([len(p) for p in kept]))
        return s
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x, x_scale = _rows(_randn((M, K), g))
        w, w_scale = _rows(0.02 * _randn((N, K), g))
        return {"case": case, "x": x, "x_scale": x_scale, "w": w, "w_scale": w_scale}
    if kind == "norm":
        M, K, act = case["M"], case["K"], DTYPE[case["act"]]
        return {"case": case, "x": _randn((M, K), g).to(act), "post": (1.0 + 0.2 * _randn((K,), g)).to(act),
                "gate": _randn((M, K), g).to(act) if case["gate"] else None,
                "residual": (3.0 * _randn((M, K), g)).to(act) if case["residual"] else None,
                "pre": (1.0 + 0.2 * _randn((K,), g)).to(act) if case["pre"] else None}
    V, Vd, act = case["V"], case["Vd"], DTYPE[case["act"]]
    news = _lengths(case)
    T = sum(news)
    logits = 2.5 * _randn((T, V), g)
    draft_logits = (logits[:, :Vd] + 0.7 * _randn((T, Vd), g)) if Vd else None
    guess = logits if draft_logits is None else draft_logits  # a draft: drawn from the draft's distribution, or a good guess
    noise = -torch.log(-torch.log(torch.rand(guess.shape, device="cuda", generator=g).clamp(1e-20, 1 - 1e-7)))
    drafts = (guess / TEMPERATURE + (noise if Vd else 0.3 * noise)).argmax(1).to(torch.int32)
    return {"case": case, "logits": logits.to(act), "draft_logits": None if draft_logits is None else draft_logits.to(act),
            "drafts": drafts, "starts": _starts(news), "u": torch.rand((T, 2), dtype=torch.float64, generator=host).cuda(),
            "temperature": torch.full((case["B"],), TEMPERATURE, dtype=torch.float32, device="cuda")}


TEMPERATURE = 0.75
SCALES = (0.75, 1.25)  # of the residual and of the block, in the norms


def _mask(parents):
    """Bit j of a token's word: it sees drafted token j of its sequence (itself and its ancestors)."""
    words = []
    for seq in parents:
        own_words = []
        for i, p in enumerate(seq):
            own_words.append((own_words[p] if p >= 0 else 0) | (1 << i))
        words += own_words
    return torch.tensor([w - (1 << 64) if w >= 1 << 63 else w for w in words], dtype=torch.int64, device="cuda")[:, None]


def _path(parents, host):
    """A path from a root down to a node."""
    at = int(torch.randint(len(parents), (1,), generator=host))
    path = []
    while at >= 0:
        path.append(at)
        at = parents[at]
    return path[::-1]


def _rows(x):
    """8-bit codes of rows and their scales."""
    s = x.abs().amax(1) / 127.0
    return torch.round(x / s[:, None]).to(torch.int8), s


# ---- one pass ----

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"step": _own_step, "verify": _own_verify, "linear": _own_linear, "norm": _own_norm, "accept": _own_accept}[kind](state)
    return {"step": _step, "verify": _verify, "linear": _linear, "norm": _norm, "accept": _accept}[kind](state)


def _own_step(s):
    from strixite_amd import kernels as kx
    if "ws" not in s:
        s["ws"] = kx.gated_delta_workspace(s["q"], s["v"], s["starts"], s["case"]["L"])
    out, _ = kx.gated_delta(s["q"], s["k"], s["v"], s["a"], s["b"], s["state"], s["starts"], s["case"]["L"], slots=s["slots"],
                            A_log=s["A_log"], dt_bias=s["dt_bias"], ws=s["ws"])
    return {"out": out, "state": s["state"]}


def _own_verify(s):
    from strixite_amd import kernels as kx
    out, u, decay, _ = kx.gated_delta_verify(s["q"], s["k"], s["v"], s["a"], s["b"], s["state"], s["starts"], s["mask"],
                                             s["case"]["L"], slots=s["slots"], A_log=s["A_log"], dt_bias=s["dt_bias"])
    kx.gated_delta_commit(s["k"], u, decay, s["state"], s["starts"], s["count"], path=s["path"], slots=s["slots"])
    return {"out": out, "state": s["state"]}


def _own_linear(s):
    from strixite_amd import ACT_BF16, ACT_F32
    from strixite_amd import kernels as kx
    if "weight" not in s:
        s["weight"] = kx.Int8Weight(s["w"], s["w_scale"])
    return kx.linear_int8(s["x"], s["x_scale"], s["weight"], out_act=ACT_F32 if s["case"]["out"] == "f32" else ACT_BF16)


def _own_norm(s):
    from strixite_amd import kernels as kx
    c = s["case"]
    y = torch.empty_like(s["x"])
    q, scale, res = kx.block_norm_int8(s["x"], post=s["post"], gate=s["gate"], residual=s["residual"], pre=s["pre"], eps=1e-6,
                                       group=c["group"] or None, gate_act=c["gate_act"], residual_scale=SCALES[0],
                                       branch_scale=SCALES[1], y=y)
    return {"q": q, "scale": scale, "y": y} if res is None else {"q": q, "scale": scale, "y": y, "residual": res}


def _own_accept(s):
    from strixite_amd import kernels as kx
    tokens, count, status = kx.mtp_accept_sampled(s["logits"], s["drafts"], s["starts"], s["u"], s["temperature"],
                                                  s["case"]["n"], draft_logits=s["draft_logits"])
    return {"tokens": tokens, "count": count, "status": status}


def _gates(s):
    """The logarithm of a token's decay, and how much of its correction it writes."""
    x = s["a"].float() + s["dt_bias"]
    g = -torch.exp(s["A_log"]) * torch.where(x > 20.0, x, torch.log1p(torch.exp(x.clamp(max=20.0))))
    return g, 1.0 / (1.0 + torch.exp(-s["b"].float()))


def _padded(s, L):
    """The sequences' rows side by side [B, heads, L, ...]; padding has keys, values, decays and corrections of zero. Also
    which places are real, and the row of each."""
    c = s["case"]
    T, dev, rep = s["q"].shape[0], s["q"].device, c["Hv"] // c["Hk"]
    first, last = s["starts"][:-1, None].long(), s["starts"][1:, None].long()
    row = first + torch.arange(L, device=dev)
    real = row < last
    row = row.clamp(max=T - 1)
    g, beta = _gates(s)
    wide = lambda x: (x.float()[row] * real[:, :, None, None]).permute(0, 2, 1, 3).contiguous()
    flat = lambda x: (x[row] * real[:, :, None]).permute(0, 2, 1).contiguous()
    unit = lambda x: x / torch.sqrt(x.square().sum(3, keepdim=True) + 1e-6)
    q = (unit(wide(s["q"])) * c["D"] ** -0.5).repeat_interleave(rep, dim=1)
    k = unit(wide(s["k"])).repeat_interleave(rep, dim=1)
    return q, k, wide(s["v"]), flat(g), flat(beta), real, row


def _inverse(A):
    """(I + A)^-1 of strict triangles (A^n = 0): the product of I + (-A)^(2^i), in 64 bits (powers can grow before they
    vanish)."""
    n = A.shape[-1]
    x = -A.double()
    one = torch.eye(n, dtype=torch.float64, device=A.device)
    inv = one + x
    for _ in range(max(0, (n - 1).bit_length() - 1)):
        x = x @ x
        inv = inv + inv @ x
    return inv.float()


def _rows_back(o, s, real, row):
    """[B, heads, L, D] to the tokens' rows; padding goes to a row of its own."""
    T = s["q"].shape[0]
    out = torch.empty((T + 1,) + (o.shape[1], o.shape[3]), dtype=torch.bfloat16, device=o.device)
    out.index_copy_(0, torch.where(real, row, T).view(-1), o.permute(0, 2, 1, 3).flatten(0, 1).to(torch.bfloat16))
    return out[:T]


def _step(s):
    """Chunks of 64: what does not need the state for all of them at once, then the state through them."""
    c = s["case"]
    C = min(64, c["L"])
    N = -(-c["L"] // C)
    q, k, v, g, beta, real, row = _padded(s, N * C)
    cut = lambda x: x.unflatten(2, (N, C)).flatten(0, 1)  # [B heads, N, C, ...]
    q, k, v, G, beta = cut(q), cut(k), cut(v), cut(g).cumsum(2), cut(beta)
    low = torch.tril(torch.ones((C, C), device=q.device)) > 0
    fade = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf))
    kT = k.transpose(2, 3).contiguous()
    inv = _inverse(torch.tril(beta[..., None] * fade * (k @ kT), -1))
    seen = fade * (q @ kT)
    kept = (torch.exp(G[..., -1:] - G)[..., None] * k).transpose(2, 3).contiguous()
    grow = torch.exp(G)[..., None]
    S = s["state"][s["slots"].long()].flatten(0, 1)
    out = torch.empty_like(v)
    for i in range(N):
        U = inv[:, i] @ (beta[:, i, :, None] * (v[:, i] - grow[:, i] * (k[:, i] @ S)))
        out[:, i] = grow[:, i] * (q[:, i] @ S) + seen[:, i] @ U
        S = grow[:, i, -1:] * S + kept[:, i] @ U
    s["state"].index_copy_(0, s["slots"].long(), S.view(c["B"], c["Hv"], c["D"], c["D"]))
    return {"out": _rows_back(out.flatten(1, 2).view(c["B"], c["Hv"], N * C, c["D"]), s, real, row), "state": s["state"]}


def _verify(s):
    """The same over one tree a sequence: a token sees its ancestors, and decays add up along its path."""
    c = s["case"]
    n = c["L"]
    q, k, v, g, beta, real, row = _padded(s, n)
    at = torch.arange(n, device=q.device)
    sees = (((s["mask"][row] >> at) & 1 == 1) & real[:, :, None])[:, None]  # [B, 1, n, n]
    G = (sees * g[:, :, None, :]).sum(3)
    fade = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~sees, -math.inf))
    kT = k.transpose(2, 3).contiguous()
    inv = _inverse(torch.tril(beta[..., None] * fade * (k @ kT), -1))
    S = s["state"][s["slots"].long()]
    grow = torch.exp(G)[..., None]
    U = inv @ (beta[..., None] * (v - grow * (k @ S)))
    out = grow * (q @ S) + (fade * (q @ kT)) @ U
    # the accepted path: entry m of it is node[m]
    keep = at < s["count"][:, None]
    node = torch.where(keep, s["path"].long(), 0)[:, None]
    pick = lambda x: torch.gather(x, 2, node[..., None].expand(-1, c["Hv"], -1, c["D"]))
    G = (g.gather(2, node.expand(-1, c["Hv"], -1)) * keep[:, None]).cumsum(2)
    kept = torch.exp(G[..., -1:] - G)[..., None] * pick(k) * keep[:, None, :, None]
    S = torch.exp(G[..., -1:])[..., None] * S + kept.transpose(2, 3).contiguous() @ pick(U)
    s["state"].index_copy_(0, s["slots"].long(), S)
    return {"out": _rows_back(out, s, real, row), "state": s["state"]}


def _linear(s):
    y = s["x"].float() @ s["w"].float().T
    return (y * s["x_scale"][:, None] * s["w_scale"]).to(DTYPE[s["case"]["out"]])


def _norm(s):
    """h = x / rms(x) * post * act(gate), r = the scaled sum with the residual, y = r / rms(r) * pre, and y as 8-bit codes.
    In 64 bits: a border decides a code."""
    c, act = s["case"], s["x"].dtype
    h = s["x"].double().view(c["M"], -1, c["group"] or c["K"])
    h = (h / torch.sqrt(h.square().mean(2, keepdim=True) + 1e-6)).flatten(1) * s["post"].double()
    if c["gate"]:
        z = s["gate"].double()
        h = h * (z if c["gate_act"] == "none" else z / (1.0 + torch.exp(-z)) if c["gate_act"] == "silu" else 1.0 / (1.0 + torch.exp(-z)))
    out = {}
    r = SCALES[1] * h
    if c["residual"]:
        out["residual"] = (SCALES[0] * s["residual"].double() + r).to(act)
        r = out["residual"].double()
    if c["pre"]:
        w = s["pre"].double()
        t = r * w
        y = t / torch.sqrt(r.square().mean(1, keepdim=True) + 1e-6)
    else:
        t = y = r
    # the codes do not depend on the root
    out["q"] = torch.round(t * 127.0 / t.abs().amax(1, keepdim=True)).to(torch.int8)
    out["scale"] = (y.abs().amax(1) / 127.0).float()
    out["y"] = y.to(act)
    return out


def _accept(s):
    """p and q in 64 bits (a border decides a token); drafts stay while u q(draft) < p(draft); then one token from what p
    has more than q, or from p behind the last draft."""
    c = s["case"]
    B, n, V = c["B"], c["n"], c["V"]
    T, dev = s["logits"].shape[0], s["logits"].device
    first, last = s["starts"][:-1].long(), s["starts"][1:].long()
    owner = torch.repeat_interleave(torch.arange(B, device=dev), last - first, output_size=T)
    temp = s["temperature"].double()[owner, None]

    def softmax(x):
        e = torch.exp((x - x.amax(1, keepdim=True)) / temp)
        return e / e.sum(1, keepdim=True)
    p = softmax(s["logits"].double())
    d = s["drafts"].long()[:, None]
    q = torch.zeros_like(p)
    if c["Vd"]:
        q[:, :c["Vd"]] = softmax(s["draft_logits"].double())
    else:
        q.scatter_(1, d, 1.0)
    stays = (s["u"][:, :1] * q.gather(1, d) < p.gather(1, d))[:, 0]
    at = torch.arange(n, device=dev)
    row = (first[:, None] + at).clamp(max=T - 1)
    is_draft = first[:, None] + at < last[:, None] - 1
    j = (stays[row] & is_draft).long().cumprod(1).sum(1)  # drafts that stay
    end = first + j
    w = torch.where((end == last - 1)[:, None], p[end], (p[end] - q[end]).clamp(min=0.0))
    total = w.cumsum(1)
    token = (total <= s["u"][end, 1:] * total[:, -1:]).sum(1).clamp(max=V - 1)
    tokens = torch.where(at < j[:, None], s["drafts"].long()[row], torch.where(at == j[:, None], token[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "count": (j + 1).to(torch.int32), "status": torch.zeros_like(j, dtype=torch.int32)}


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind in ("step", "verify"):
        B, L, Hk, Hv, D = (case[x] for x in ("B", "L", "Hk", "Hv", "D"))
        T = sum(_lengths(case))
        rows = T * (2 * D * (2 * Hk + 2 * Hv) + 4 * Hv)  # q, k, v, out and the gates
        if kind == "step":
            return {"bytes": rows + 8 * B * Hv * D * D, "flops": 6 * T * Hv * D * D}
        kept = T // 2
        return {"bytes": rows + 12 * B * Hv * D * D + 4 * Hv * D * (T + kept) + 2 * kept * Hk * D,
                "flops": (4 * T + 2 * kept) * Hv * D * D + 4 * T * L * Hv * D}
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K + 4 * N + M * K + 4 * M + M * N * (4 if case["out"] == "f32" else 2), "flops": 2 * M * N * K}
    if kind == "norm":
        M, K, e = case["M"], case["K"], 4 if case["act"] == "f32" else 2
        arrays = 2 + (1 if case["gate"] else 0) + (2 if case["residual"] else 0)
        return {"bytes": M * K * (e * arrays + 1) + 4 * M + K * e * (2 if case["pre"] else 1), "flops": 12 * M * K}
    T, e = sum(_lengths(case)), 4 if case["act"] == "f32" else 2
    drafted = T - case["B"]
    return {"bytes": e * (T * case["V"] + drafted * case["Vd"]) + 20 * T, "flops": 4 * (T * case["V"] + drafted * case["Vd"])}


# ---- the same results in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        x = s["x"].double() * s["x_scale"].double()[:, None]
        parts = [x @ (s["w"][r:r + 1024].double() * s["w_scale"][r:r + 1024, None].double()).T for r in range(0, case["N"], 1024)]
        return torch.cat(parts, dim=1)
    if kind == "norm":
        return _exact_norm(case, s)
    if kind == "accept":
        return _exact_accept(case, s)
    return _exact_delta(case, s)


def _exact_norm(case, s):
    x = s["x"].double()
    group = case["group"] or case["K"]
    h = torch.cat([p / (p.pow(2).sum(1, keepdim=True) / group + 1e-6).sqrt() for p in x.split(group, dim=1)], dim=1)
    h = h * s["post"].double()[None]
    if case["gate"]:
        z = s["gate"].double()
        h = h * {"none": z, "silu": z * torch.sigmoid(z), "sigmoid": torch.sigmoid(z)}[case["gate_act"]]
    r = h * SCALES[1]
    out = {"q": None}
    if case["residual"]:
        r = r + s["residual"].double() * SCALES[0]
        out["residual"] = r
        r = r.float().to(s["x"].dtype).double()  # the stream keeps what is stored
    if case["pre"]:
        r = r * s["pre"].double()[None] / (r.pow(2).sum(1, keepdim=True) / case["K"] + 1e-6).sqrt()
    return {**out, "scale": r.abs().max(1).values / 127.0, "y": r}


def _exact_accept(case, s):
    """Sequence by sequence, row by row: a row behind the first draft that falls is not looked at."""
    starts = s["starts"].tolist()
    tokens, count = torch.full((case["B"], case["n"]), -1, dtype=torch.int32), []
    for b in range(case["B"]):
        t, end = starts[b], starts[b + 1] - 1
        while True:
            p = torch.softmax(s["logits"][t].double() / s["temperature"][b].double(), dim=0)
            if t == end:
                w = p
                break
            d, q = int(s["drafts"][t]), torch.zeros_like(p)
            if case["Vd"]:
                q[:case["Vd"]] = torch.softmax(s["draft_logits"][t].double() / s["temperature"][b].double(), dim=0)
            else:
                q[d] = 1.0
            if not float(s["u"][t, 0]) * float(q[d]) < float(p[d]):
                w = (p - q).clamp(min=0.0)
                break
            tokens[b, t - starts[b]] = d
            t += 1
        run_to = torch.cumsum(w, dim=0)
        tokens[b, t - starts[b]] = int(torch.searchsorted(run_to, s["u"][t, 1] * run_to[-1], right=True))
        count.append(t - starts[b] + 1)
    return {"tokens": tokens.cuda(), "count": _i32(count), "status": torch.zeros(case["B"], dtype=torch.int32, device="cuda")}


def _exact_delta(case, s):
    """Token by token; a drafted token goes on from its parent's state."""
    Hk, Hv, D = case["Hk"], case["Hv"], case["D"]
    starts, slots = s["starts"].tolist(), s["slots"].tolist()
    state = s["state"].double()
    a = s["a"].double() + s["dt_bias"].double()
    alpha = torch.exp(-s["A_log"].double().exp() * torch.nn.functional.softplus(a))
    beta = torch.sigmoid(s["b"].double())
    unit = lambda x: x / (x.pow(2).sum(2, keepdim=True) + 1e-6).sqrt()
    q = unit(s["q"].double()) / math.sqrt(D)
    k = unit(s["k"].double())
    v = s["v"].double()
    out = torch.zeros((starts[-1], Hv, D), dtype=torch.float64, device="cuda")
    spread = lambda x: x[:, None].expand(Hk, Hv // Hk, D).reshape(Hv, D)
    for b, slot in enumerate(slots):
        S, nodes = state[slot], []
        for t in range(starts[b], starts[b + 1]):
            i = t - starts[b]
            if case["kind"] == "verify":
                word = int(s["mask"][t, 0]) & ((1 << i) - 1)
                S = nodes[word.bit_length() - 1] if word else state[slot]  # the newest ancestor is the parent
            kt = spread(k[t])
            S = S * alpha[t][:, None, None]
            u = (v[t] - (S * kt[:, :, None]).sum(1)) * beta[t][:, None]
            S = S + kt[:, :, None] * u[:, None, :]
            out[t] = (S * spread(q[t])[:, :, None]).sum(1)
            if case["kind"] == "verify":
                nodes.append(S)
        if case["kind"] == "verify":
            S = nodes[int(s["path"][b, int(s["count"][b]) - 1])]
        state[slot] = S
    return {"out": out, "state": state}
