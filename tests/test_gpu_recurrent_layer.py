"""The recurrent layer's operators as a verify runs them: VerifyDelta against a plain layer in 64 bits, drafted and accepted tokens
against the same tokens decoded one by one, acceptance deciding what is committed, streams and a replayed graph.

The layer's 8-bit codes are the plain layer's own steps, so both are compared behind each rounding: the plain layer takes the
kernel's codes where it makes them, and the projections, the rule and the norms behind them are held to their own tolerances
(u16 = 2^-8 of BF16, and 2^-16 of a sum of absolute products for what precedes it)."""
import pytest
import torch

from strixite_amd import SxError
from strixite_amd import kernels as kx
from strixite_amd import synthetic as syn
from strixite_amd.verify import VerifyDelta, VerifyTail

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -8
BF = torch.bfloat16
d, Hk, Hv, Dk, Dv = 256, 2, 4, 64, 64


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def int8(N, K, g):
    w = 0.06 * torch.randn(N, K, device="cuda", generator=g)
    s = w.abs().amax(1) / 127
    return kx.Int8Weight(torch.round(w / s[:, None]).to(torch.int8), s)


def layer(seed=0, max_tokens=64, **kw):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return VerifyDelta((1 + 0.2 * r(d)).to(BF), int8(2 * Hk * Dk + 2 * Hv * Dv + 2 * Hv, d, g), torch.log(1 + 15 * torch.rand(Hv, device="cuda", generator=g)),
                       -3 + r(Hv), (1 + 0.2 * r(Dv)).to(BF), int8(d, Hv * Dv, g), Hk, Hv, Dk, Dv, max_tokens, **kw)


def near(got, want, tol):
    assert torch.isfinite(got).all() and (got.double() - want.double()).norm() <= tol * want.double().norm(), float((got.double() - want.double()).norm() / want.double().norm())


def plain(L, x, residual, state, parents):
    """One sequence through the layer in 64 bits from the kernels' codes: y, the residual, the state behind each token."""
    D = lambda t: t.double()
    r = x if residual is None else (L.residual_scale * D(residual) + D(x) / (D(x).square().mean(1, keepdim=True) + L.eps).sqrt() * D(L.post_w)).to(BF)
    rows = (D(L.q8[:x.shape[0]]) * D(L.scale[:x.shape[0]])[:, None]) @ (D(L.proj.q) * D(L.proj.scale)[:, None]).T
    T = x.shape[0]
    near(L.rows[:T], rows, U16)
    rows = D(L.rows[:T])
    y = D(r) / (D(r).square().mean(1, keepdim=True) + L.eps).sqrt() * D(L.norm_w)
    near(D(L.q8[:T]) * D(L.scale[:T])[:, None], y, 0.02)  # codes of 127 steps a side: 1 / (127 sqrt(12)) of the largest, a few times the mean
    q, k, v, z, a, b = rows.split([Hk * Dk, Hk * Dk, Hv * Dv, Hv * Dv, Hv, Hv], dim=1)
    unit = lambda t: t / (t.square().sum(2, keepdim=True) + 1e-6).sqrt()
    q, k = (unit(t.reshape(T, Hk, Dk)).repeat_interleave(Hv // Hk, 1) for t in (q, k))
    v = v.reshape(T, Hv, Dv)
    al = torch.exp(-D(L.A_log).exp() * torch.nn.functional.softplus(a + D(L.dt_bias)))
    be = torch.sigmoid(b)
    nodes, out = [], torch.zeros(T, Hv, Dv, dtype=torch.float64, device="cuda")
    for t in range(T):
        S = (D(state) if parents[t] < 0 else nodes[parents[t]]) * al[t][:, None, None]
        u = be[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
        S = S + k[t][:, :, None] * u[:, None]
        out[t] = (S * q[t][:, :, None]).sum(1) * Dk ** -0.5
        nodes.append(S)
    near(L.out[:T], out, U16)
    o = D(L.out[:T])
    o = (o / (o.square().mean(2, keepdim=True) + L.eps).sqrt() * D(L.head_w)).flatten(1) * z * torch.sigmoid(z)
    near(D(L.o8[:T]) * D(L.o_scale[:T])[:, None], o, 0.03)
    want = (D(L.o8[:T]) * D(L.o_scale[:T])[:, None]) @ (D(L.out_w.q) * D(L.out_w.scale)[:, None]).T
    return want, r, nodes


@pytest.mark.parametrize("post", [False, True])
def test_a_layer_against_the_plain_one(post):
    g = gen(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    L = layer(1, post_w=(1 + 0.2 * r(d)).to(BF) if post else None, residual_scale=0.5 if post else 1.0)
    if not post:
        L.post_w = None
    T, parents = 9, [-1, 0, 0, 1, 3, 2, 5, 5, 6]
    x, residual = r(T, d).to(BF), (2 * r(T, d)).to(BF) if post else None
    state = 0.4 * r(3, Hv, Dk, Dv)
    before, slots, starts, mask = state.clone(), i32([2]), i32([0, T]), kx.tree_mask([parents]).cuda()
    y, res = L.forward(x, residual, state, starts, T, mask=mask, slots=slots)
    want, r2, nodes = plain(L, x, residual, before[2], parents)
    near(y, want, U16)
    assert torch.equal(res, r2) and torch.equal(state, before) and int(L.err[0]) == 0
    L.commit(state, starts, i32([4]), path=i32([[0, 2, 5, 6]]), slots=slots)
    near(state[2], nodes[6], 40 * 2.0 ** -24)
    assert torch.equal(state[:2], before[:2])


def test_verifies_go_where_decoding_goes():
    """Prompt, then five verifies whose accepted prefixes are committed: the states are those of the same tokens decoded one by one."""
    L, one = layer(2, max_tokens=256), layer(2, max_tokens=256)
    g = gen(7)
    B, lens = 2, [100, 33]
    a, b = torch.zeros(B, Hv, Dk, Dv, device="cuda"), torch.zeros(B, Hv, Dk, Dv, device="cuda")
    x = torch.randn(sum(lens), d, device="cuda", generator=g).to(BF)
    starts = i32([0, lens[0], sum(lens)])
    ya, _ = L.forward(x, None, a, starts, 100)
    for i in range(B):  # the same prompts in pieces
        lo = 0
        while lo < lens[i]:
            hi = min(lo + 16, lens[i])
            first = sum(lens[:i]) + lo
            yb, _ = one.forward(x[first:first + hi - lo], None, b, i32([0, hi - lo]), 16, slots=i32([i]))
            # the out codes' steps: a value at a border falls to either side, one step of 254 of its row
            near(yb, ya[first:first + hi - lo], 0.01)
            lo = hi
    near(a, b, 100 * 2.0 ** -24)
    for step in range(5):
        n = 6
        x = torch.randn(B * n, d, device="cuda", generator=g).to(BF)
        mask = kx.tree_mask([list(range(-1, n - 1))] * B).cuda()
        count = [1 + (step + i) % n for i in range(B)]
        L.forward(x, None, a, i32([0, n, 2 * n]), n, mask=mask)
        L.commit(a, i32([0, n, 2 * n]), i32(count), max_count=n)
        for t in range(max(count)):
            on = [i for i in range(B) if t < count[i]]
            one.forward(torch.cat([x[i * n + t:i * n + t + 1] for i in on]), None, b, i32(list(range(len(on) + 1))), 1, slots=i32(on))
        near(a, b, 200 * 2.0 ** -24)


def test_there_is_nothing_to_commit_behind_a_prompt():
    L = layer(2)
    x, state = torch.randn(8, d, device="cuda").to(BF), torch.zeros(1, Hv, Dk, Dv, device="cuda")
    L.forward(x, None, state, i32([0, 8]), 8)
    with pytest.raises(SxError, match="no drafted tokens"):
        L.commit(state, i32([0, 8]), i32([1]), max_count=8)


def test_what_is_accepted_is_committed():
    """Head, acceptance and commit with nothing read back in between, captured and replayed."""
    L = layer(3)
    g = gen(11)
    B, n, V = 3, 5, 900
    tail = VerifyTail(syn.qweight(8, V, d, 64, seed=5), V, 20, B * n)
    state0 = 0.3 * torch.randn(B, Hv, Dk, Dv, device="cuda", generator=g)
    x = torch.randn(B * n, d, device="cuda", generator=g).to(BF)
    starts, mask = i32([0, n, 2 * n, 3 * n]), kx.tree_mask([list(range(-1, n - 1))] * B).cuda()
    temperature = torch.tensor([1.0, 0.0, 0.7], device="cuda")
    u = torch.rand(B * n, 2, dtype=torch.float64, device="cuda", generator=g)
    draft_logits = torch.randn(B * n, V, device="cuda", generator=g)
    drafts = draft_logits.argmax(1).to(torch.int32)

    def step(state):
        y, _ = L.forward(x, None, state, starts, n, mask=mask)
        tokens, count, status = tail.accept_sampled(y, drafts, starts, u, temperature, n, draft_logits=draft_logits)
        L.commit(state, starts, count, max_count=n)
        return tokens, count, status
    s = state0.clone()
    tokens, count, status = step(s)
    assert status.tolist() == [0, 0, 0] and all(1 <= c <= n for c in count.tolist())
    ref = state0.clone()
    y, _ = L.forward(x, None, ref, starts, n, mask=mask)
    L.commit(ref, starts, count, max_count=n)
    assert torch.equal(s, ref) and not torch.equal(ref, state0)
    live = state0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(live)
    eager = state0.clone()
    for i in range(4):
        u.copy_(torch.rand(B * n, 2, dtype=torch.float64, device="cuda", generator=gen(i)))
        drafts.copy_(torch.randint(0, V, (B * n,), device="cuda", generator=gen(i)).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        assert all(torch.equal(p, q) for p, q in zip(outs, want)) and torch.equal(live, eager)


def test_forwards_on_two_streams():
    L = layer(4, mix=lambda q, k, v: (q.mul_(0.5), v.add_(0.25)))
    g = gen(13)
    x = [torch.randn(6, d, device="cuda", generator=g).to(BF) for _ in range(2)]
    state = 0.3 * torch.randn(1, Hv, Dk, Dv, device="cuda", generator=g)
    starts, mask = i32([0, 6]), kx.tree_mask([list(range(-1, 5))]).cuda()
    refs = [L.forward(t, None, state, starts, 6, mask=mask)[0].clone() for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    for _ in range(5):
        ys = [L.forward(t, None, state, starts, 6, mask=mask, stream=s)[0] for t, s in zip(x, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ys, refs))
