"""The gated delta rule on cuda:0 against the rule itself, token by token in 64 bits.

Tolerances, u16 = 2^-8 (BF16, half a step), u32 = 2^-24. With keys of length one, 0 <= beta <= 1 and decays up to 1 a step is a
contraction of the state's columns, so a step's rounding is not amplified: with c the roundings of a step,
  e <- alpha e + c u32 (|S| + |u| + |v|) per column (2-norms), c = Dk + 24 + 8 |g| (a sum of Dk products, the gates' exponentials, the
  update); in chunks of 64 another 64^2: the rows of (I + A)^-1, entries of at most one, are sums of up to 64 products of such sums.
  out: u16 |o| + scale |q| (e + (Dk + c) u32 |S|).
That is a worst case. Roundings are random: the 2-norm of all errors over the result's is held to 40 u32 for states, corrections
and u16 for outputs (a sum of 128 products is off by 6 u32 of its norm, and a few such sums meet in a state).
"""
import math

import numpy as np
import pytest
import torch

from strixite_amd import SxError
from strixite_amd import kernels as kx

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -8, 2.0 ** -24
BF = torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Tokens:
    def __init__(self, lens, Hk=2, Hv=4, Dk=128, Dv=128, seed=0, raw=False, f32=False, normalize=True, slots=True, spare=0, strong=False):
        g, host = gen(seed), torch.Generator().manual_seed(seed)
        self.lens, self.Hk, self.Hv, self.Dk, self.Dv, self.normalize = lens, Hk, Hv, Dk, Dv, normalize
        B, self.T = len(lens), sum(lens)
        rows = max(self.T + spare, 1)
        self.starts, self.max_len = i32([0] + np.cumsum(lens).tolist()), max(max(lens), 1)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        if Dk == Dv:  # slices of one projection
            qkv = r(rows, 2 * Hk + Hv, Dk).to(BF)
            self.q, self.k, self.v = qkv.split([Hk, Hk, Hv], dim=1)
        else:
            self.q, self.k, self.v = r(rows, Hk, Dk).to(BF), r(rows, Hk, Dk).to(BF), r(rows, Hv, Dv).to(BF)
        if strong:  # keys that are all alike: the triangle's entries are near one
            self.k.copy_((1.0 + 0.1 * r(rows, Hk, Dk)).to(BF))
        if not normalize:
            self.k.mul_(0.9 / math.sqrt(Dk)), self.q.mul_(0.9 / math.sqrt(Dk))
            self.k.div_(self.k.float().norm(dim=2, keepdim=True).clamp(min=1.0).to(BF) * 1.02)
        dt = torch.float32 if f32 else BF
        if raw:
            self.a, self.b = (-0.3 * torch.rand(rows, Hv, device="cuda", generator=g)).to(dt), torch.rand(rows, Hv, device="cuda", generator=g).to(dt)
            self.A_log = self.dt_bias = None
        else:
            both = r(rows, 2 * Hv).to(dt)
            self.a, self.b = both[:, :Hv], both[:, Hv:]
            self.A_log, self.dt_bias = torch.log(1 + 15 * torch.rand(Hv, device="cuda", generator=g)), -3 + r(Hv)
        states = B + 3 if slots else B
        self.state = 0.5 * r(states, Hv, Dk, Dv)
        self.slots = torch.randperm(states, generator=host)[:B].to(torch.int32).cuda() if slots else None
        self.host = host

    def slot(self, b):
        return b if self.slots is None else int(self.slots[b])

    def kw(self, **kw):
        return {**dict(slots=self.slots, A_log=self.A_log, dt_bias=self.dt_bias, normalize=self.normalize), **kw}

    def run(self, state, **kw):
        return kx.gated_delta(self.q, self.k, self.v, self.a, self.b, state, self.starts, kw.pop("max_len", self.max_len), **self.kw(**kw))

    def verify(self, state, mask, **kw):
        return kx.gated_delta_verify(self.q, self.k, self.v, self.a, self.b, state, self.starts, mask, self.max_len, **self.kw(**kw))

    def gates(self):
        a, b = self.a.double(), self.b.double()
        if self.A_log is None:
            return a, b
        return -self.A_log.double().exp() * torch.nn.functional.softplus(a + self.dt_bias.double()), torch.sigmoid(b)

    def rule(self, parents=None, chunked=False):
        """out, states, u / |k|, g, and the tolerances of out and states; parents: each sequence's tree (None: chains)."""
        unit = lambda x: x / (x.pow(2).sum(2, keepdim=True) + 1e-6).sqrt() if self.normalize else x
        rep = self.Hv // self.Hk
        kl = ((self.k.double().pow(2).sum(2) + 1e-6).sqrt() if self.normalize else torch.ones_like(self.k[..., 0].double()))
        q = unit(self.q.double()).repeat_interleave(rep, 1) / math.sqrt(self.Dk)
        k, v = unit(self.k.double()).repeat_interleave(rep, 1), self.v.double()
        g, beta = self.gates()
        out, tol = torch.zeros(self.T, self.Hv, self.Dv, dtype=torch.float64, device="cuda"), torch.zeros(self.T, self.Hv, self.Dv, dtype=torch.float64, device="cuda")
        us = torch.zeros_like(out)
        state, stol = self.state.double(), torch.zeros_like(self.state, dtype=torch.float64)
        self.nodes = []
        t0 = 0
        for b, n in enumerate(self.lens):
            S0, nodes = state[self.slot(b)].clone(), []
            e0 = torch.zeros(self.Hv, self.Dv, dtype=torch.float64, device="cuda")
            for i in range(n):
                t = t0 + i
                par = i - 1 if parents is None else parents[b][i]
                S, e = (S0, e0) if par < 0 else nodes[par]
                al = g[t].exp()[:, None]
                S = S * al[:, :, None]
                u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
                c = (self.Dk + 24 + 8 * g[t].abs())[:, None] + (64 ** 2 if chunked else 0)
                e = al * e + c * U32 * (S.norm(dim=1) + u.abs() + v[t].abs())
                S = S + k[t][:, :, None] * u[:, None, :]
                out[t] = (S * q[t][:, :, None]).sum(1)
                tol[t] = U16 * out[t].abs() + q[t].norm(dim=1)[:, None] * (e + (self.Dk + c) * U32 * S.norm(dim=1)) + 1e-30
                us[t] = u / kl[t].repeat_interleave(rep)[:, None]
                nodes.append((S, e))
            if n and parents is None:
                state[self.slot(b)], stol[self.slot(b)] = nodes[-1][0], nodes[-1][1][:, None, :]
            self.nodes.append(nodes)
            t0 += n
        return out, state, us, g, tol, stol


def close(got, ref, tol, rms, what=""):
    d = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (d <= tol).all(), (what, float((d - tol).max()), float((d / tol.clamp(min=1e-300)).max()))
    assert d.norm() <= rms * ref.norm() + 1e-30, (what, float(d.norm() / ref.norm()))


CASES = [  # lens, heads and dims, more
    ([1], {}), ([1, 0, 1, 1], dict(Hk=1, Hv=3)), ([16, 3, 0, 7], dict(Dk=64, Dv=64)), ([5], dict(raw=True, f32=True, slots=False)),
    ([2, 16], dict(Dv=48, Hk=2, Hv=2)), ([9, 1], dict(normalize=False, raw=True)), ([16] * 5, dict(strong=True)),
    ([17], {}), ([64], dict(slots=False)), ([65, 0, 1], dict(Hk=1, Hv=2)), ([63, 130, 16], dict(Dk=64, Dv=64, Hk=2, Hv=6)),
    ([200, 33], dict(Dv=16, raw=True)), ([129], dict(Dv=256, Hk=1, Hv=1, f32=True)), ([70, 90], dict(normalize=False, raw=True, f32=True)),
    ([320, 64, 128, 1], dict(Dk=64, Dv=128, Hk=3, Hv=3)), ([130, 64], dict(strong=True, raw=True)), ([257, 19], dict(Dk=128, Dv=80)),
]


@pytest.mark.parametrize("lens,more", CASES)
def test_sequences(lens, more):
    x = Tokens(lens, seed=len(lens) + max(lens), **more)
    chunked = x.max_len > 16
    out, state, _, _, tol, stol = x.rule(chunked=chunked)
    got = x.state.clone()
    o, err = x.run(got, err=torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert err.tolist()[0] == 0
    close(o, out, tol, U16, "out")
    used = [x.slot(b) for b, n in enumerate(lens) if n]
    close(got[used], state[used], stol[used], 40 * U32, "state")
    rest = [i for i in range(got.shape[0]) if i not in used]
    assert torch.equal(got[rest], x.state[rest])  # nobody else's
    if not chunked:  # the same tokens as chunks: the limit chooses, not the lengths
        again = x.state.clone()
        o, _ = x.run(again, max_len=64)
        _, _, _, _, tol, stol = x.rule(chunked=True)
        close(o, out, tol, U16, "out")
        close(again[used], state[used], stol[used], 40 * U32, "state")


@pytest.mark.parametrize("cut", [64, 100, 1])
def test_a_prompt_in_two_calls(cut):
    x = Tokens([230], seed=3)
    out, state, _, _, tol, stol = x.rule(chunked=True)
    got, o = x.state.clone(), torch.empty(230, x.Hv, x.Dv, dtype=BF, device="cuda")
    for lo, hi in ((0, cut), (cut, 230)):
        part = lambda t: t[lo:hi]
        kx.gated_delta(part(x.q), part(x.k), part(x.v), part(x.a), part(x.b), got, i32([0, hi - lo]), hi - lo, **x.kw(out=o[lo:hi]))
    close(o, out, tol, U16)
    close(got[x.slot(0)], state[x.slot(0)], stol[x.slot(0)], 40 * U32)


def test_heads_ahead_of_tokens_and_a_single_row_of_stride_zero():
    """[heads, tokens, dim] in memory on every side, and an output of one token whose stride says nothing."""
    x = Tokens([70, 20], Hk=2, Hv=4, seed=12)
    s = x.state.clone()
    ref, _ = x.run(s)
    turn = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    x.q, x.k, x.v = turn(x.q), turn(x.k), turn(x.v)
    got, out = x.state.clone(), torch.empty(x.Hv, x.T, x.Dv, dtype=BF, device="cuda").transpose(0, 1)
    x.run(got, out=out)
    assert torch.equal(out, ref) and torch.equal(got, s)
    x = Tokens([1], seed=13)
    for limit in (1, 64):
        a, b = x.state.clone(), x.state.clone()
        ref, _ = x.run(a, max_len=limit)
        out = torch.zeros(1, x.Hv, x.Dv, dtype=BF, device="cuda").as_strided((1, x.Hv, x.Dv), (0, x.Dv, 1))
        x.run(b, max_len=limit, out=out)
        assert torch.equal(out, ref) and torch.equal(a, b)


def test_new_sequences_long_decays_and_full_resets():
    x = Tokens([40, 90, 6], raw=True, f32=True, seed=5)
    x.state.zero_()
    x.a[10] = -math.inf   # forgets everything
    x.a[50:60] = -90.0    # sums far past what FP32 exponentials reach
    x.a[60:65] = 0.0      # and nothing
    out, state, _, _, tol, stol = x.rule(chunked=True)
    tol[x.a[:, :, None].expand_as(tol) == -math.inf] += 1e-6
    got = x.state.clone()
    o, _ = x.run(got)
    fin = torch.isfinite(tol)
    close(torch.where(fin, o.double(), out), out, torch.where(fin, tol, torch.ones_like(tol)), U16)
    assert torch.isfinite(got).all() and (got.double() - state).norm() <= 40 * U32 * state.norm()


def tree(n, host, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] * n
    return [int(torch.randint(max(-1, i - 6), i, (1,), generator=host)) if i else -1 for i in range(n)]


def paths(parents, host):
    out = []
    for p in parents:
        path, at = [], int(torch.randint(len(p), (1,), generator=host)) if p else -1
        while at >= 0:
            path.append(at)
            at = p[at]
        out.append(path[::-1])
    return out


@pytest.mark.parametrize("lens,kind,more", [
    ([1], "chain", {}), ([6], "chain", dict(Hk=1, Hv=2)), ([16, 0, 5], "tree", dict(Dk=64, Dv=64)), ([17, 3], "tree", {}),
    ([24] * 9, "tree", dict(Hk=4, Hv=16)), ([32, 31, 0, 1], "star", dict(Dv=80)), ([33], "tree", {}), ([64, 1, 50], "chain", dict(Dk=64, Dv=48)),
    ([64, 40], "tree", dict(raw=True, f32=True, normalize=False)), ([64] * 20, "tree", dict(Hk=4, Hv=8, Dv=64)), ([12], "chain", dict(strong=True)),
])
def test_verify_and_commit(lens, kind, more):
    x = Tokens(lens, seed=sum(lens), **more)
    parents = [tree(n, x.host, kind) for n in lens]
    mask = kx.tree_mask(parents).cuda()
    out, _, us, g, tol, _ = x.rule(parents)
    before = x.state.clone()
    o, u, decay, _ = x.verify(x.state, mask)
    assert torch.equal(before, x.state)
    # P U: two BF16 terms of each, 2^-16 of sums |P||u| <= sum |u| scale
    close(o, out, tol + 2.0 ** -14 * us.abs().max() * 12 * x.Dk ** -0.5, U16, "out")
    assert (u.double() - us).norm() <= 40 * U32 * us.norm()
    assert (decay.double() - g[:x.T]).abs().max() <= 8 * U32 * g.abs().max()
    path = paths(parents, x.host)
    counts = [len(p) for p in path]
    padded = torch.zeros(len(lens), max(counts + [1]) + 2, dtype=torch.int32)
    for b, p in enumerate(path):
        padded[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    kx.gated_delta_commit(x.k, u, decay, x.state, x.starts, i32(counts), path=padded.cuda(), slots=x.slots, err=err)
    assert err.tolist()[0] == 0
    for b, p in enumerate(path):
        want, e = x.nodes[b][p[-1]] if p else (before[x.slot(b)].double(), torch.zeros(1, device="cuda"))
        got = x.state[x.slot(b)]
        assert (got.double() - want).norm() <= 40 * U32 * want.norm()
        if not p:
            assert torch.equal(got, before[x.slot(b)])
    rest = [i for i in range(before.shape[0]) if i not in [x.slot(b) for b in range(len(lens))]]
    assert torch.equal(x.state[rest], before[rest])


def test_a_chains_commit_is_the_steps_state():
    """verify + commit of a prefix (no path) against the steps that decoding would take."""
    x = Tokens([9, 4, 16], seed=8)
    mask = kx.tree_mask([list(range(-1, n - 1)) for n in x.lens]).cuda()
    a, b = x.state.clone(), x.state.clone()
    o, u, decay, _ = x.verify(a, mask)
    ref, _ = x.run(b)
    assert (o.double() - ref.double()).norm() <= 2 * U16 * ref.double().norm()
    kx.gated_delta_commit(x.k, u, decay, a, x.starts, i32([9, 4, 16]), max_count=16, slots=x.slots)
    assert (a.double() - b.double()).norm() <= 40 * U32 * b.double().norm()


def test_commit_of_all_layers_at_once():
    layers = [Tokens([6, 0, 3], Hk=1, Hv=2, Dk=64, Dv=64, seed=s) for s in range(3)]
    mask = kx.tree_mask([list(range(-1, 5)), [], list(range(-1, 2))]).cuda()
    outs = [x.verify(x.state, mask) for x in layers]
    k, u, decay = (torch.stack(t) for t in ([x.k for x in layers], [o[1] for o in outs], [o[2] for o in outs]))
    state, slots = torch.stack([x.state for x in layers]), layers[0].slots
    want = state.clone()
    count = i32([4, 0, 3])
    for i in range(3):
        kx.gated_delta_commit(k[i], u[i], decay[i], want[i], layers[0].starts, count, max_count=8, slots=slots)
    kx.gated_delta_commit(k, u, decay, state, layers[0].starts, count, max_count=8, slots=slots)
    assert torch.equal(state, want)


# ---------------- what must not spread ----------------

def test_rows_behind_the_last_sequence_stay():
    for lens in ([5, 2], [70, 2]):
        x = Tokens(lens, seed=1, spare=9)
        for t in (x.q, x.k, x.v):
            t[x.T:] = math.nan
        out = torch.full((x.T + 9, x.Hv, x.Dv), 7.0, dtype=BF, device="cuda")
        o, _ = x.run(x.state.clone(), out=out)
        assert (o[x.T:] == 7).all() and torch.isfinite(o[:x.T]).all()


@pytest.mark.parametrize("n,at", [(12, 5), (100, 70), (100, 3), (64, 63)])
@pytest.mark.parametrize("what", ["k", "q", "v", "a"])
def test_a_token_that_is_no_number(n, at, what):
    """Tokens before it, other heads and other sequences are as without it; those from it on are NaN (q: its own row; v: its column)."""
    x = Tokens([n, n], Hk=2, Hv=4, seed=n)
    clean, cs = x.state.clone(), x.state.clone()
    ref, _ = x.run(cs)
    t = getattr(x, what)
    t[at, 0] = math.nan  # of the first head: value heads 0 and 1 where it is a key head
    if what == "v":
        t[at, 0] = x.v[at, 1]
        t[at, 0, 5] = math.inf
    heads = {"k": 2, "q": 2, "v": 1, "a": 1}[what]
    o, _ = x.run(clean)
    assert torch.equal(o[:at], ref[:at]) and torch.equal(o[n:], ref[n:]) and torch.equal(o[:, heads:], ref[:, heads:])
    assert torch.equal(clean[:, heads:], cs[:, heads:])  # value heads that share the key head, too
    if what == "q":
        assert o[at, :heads].isnan().all() and torch.equal(o[at + 1:], ref[at + 1:]) and torch.equal(clean, cs)
    elif what == "v":
        assert o[at:n, 0, 5].isnan().all() or not torch.isfinite(o[at:n, 0, 5]).any()
        assert torch.isfinite(o[:n, 0, 6:]).all() and not torch.isfinite(clean[x.slot(0), 0, :, 5]).any()
    else:
        assert not torch.isfinite(o[at:n, :heads]).any() and not torch.isfinite(clean[x.slot(0), :heads]).any()
        assert torch.equal(clean[x.slot(1)], cs[x.slot(1)])


def test_a_drafted_token_touches_only_those_that_see_it():
    x = Tokens([40], seed=2)
    parents = [tree(40, x.host, "tree")]
    parents[0][30] = 12
    mask = kx.tree_mask(parents).cuda()
    ref, u0, g0, _ = x.verify(x.state, mask)
    x.k[12] = math.nan
    o, u, _, _ = x.verify(x.state, mask)
    sees = torch.tensor([bool(int(m) >> 12 & 1) for m in mask[:, 0].cpu()], device="cuda")
    assert sees[12] and sees[30] and not sees.all()
    assert torch.equal(u[~sees], u0[~sees]) and o[sees].isnan().all()
    d = (o[~sees].double() - ref[~sees].double()).abs()  # P U in FP32 there
    assert (d <= 2 * U16 * ref[~sees].double().abs() + 1e-2 * U16).all()


def test_impossible_words_on_the_device():
    err = lambda: torch.zeros(4, dtype=torch.int32, device="cuda")
    for lens in ([5, 6, 7], [70, 6, 7]):
        x = Tokens(lens, seed=4)
        clean = x.state.clone()
        ref, _ = x.run(clean)
        mask = kx.tree_mask([list(range(-1, min(n, 64) - 1)) for n in lens]).cuda()
        good = x.slots.clone()
        # a slot that is none, and one that two have
        for bad, nan in ((good.clone().index_fill_(0, i32([1]).long(), 99), [1]), (torch.stack([good[0], good[1], good[1]]), [1, 2])):
            x.slots, s, e = bad, x.state.clone(), err()
            o, _ = x.run(s, err=e)
            at = np.cumsum([0] + lens)
            for b in range(3):
                rows = o[at[b]:at[b + 1]]
                assert rows.isnan().all() if b in nan else torch.equal(rows, ref[at[b]:at[b + 1]])
            assert e[0] == 1 and int(e[2]) in nan
            keep = [int(i) for i in range(s.shape[0]) if i != int(good[0]) and not (len(nan) == 1 and i == int(good[2]))]
            assert torch.equal(s[keep], x.state[keep])
        x.slots = good
        # runs of tokens that cannot be: none of theirs is touched
        for starts in ([0, -3, 11, 18], [0, 5, 3, 18], [0, 5, 11, 10 ** 6]):
            if lens[0] != 5:
                continue
            s, e = x.state.clone(), err()
            out = torch.full((x.T, x.Hv, x.Dv), 7.0, dtype=BF, device="cuda")
            kx.gated_delta(x.q, x.k, x.v, x.a, x.b, s, i32(starts), 7, **x.kw(out=out, err=e))
            assert e[0] == 1 and torch.isfinite(out).all()
        if lens[0] == 5:
            o, u, g, e = x.verify(x.state, mask, err=err())
            for kw, b in ((dict(count=i32([6, 1, 1])), 0), (dict(count=i32([1, -1, 1])), 1),
                          (dict(count=i32([1, 1, 2]), path=i32([[0, 0], [0, 0], [0, 7]])), 2), (dict(count=i32([1, 9, 1]), max_count=8), 1)):
                s, e = x.state.clone(), err()
                kx.gated_delta_commit(x.k, u, g, s, x.starts, slots=x.slots, err=e, **{**(dict(max_count=8) if "path" not in kw else {}), **kw})
                assert e[0] == 1 and e[2] == b and torch.equal(s[x.slot(b)], x.state[x.slot(b)])
                assert not torch.equal(s[x.slot((b + 1) % 3)], x.state[x.slot((b + 1) % 3)])


def test_empty_sequences_may_share_a_slot():
    x = Tokens([3, 0, 0], seed=6)
    x.slots = torch.stack([x.slots[0], x.slots[0], torch.tensor(-1, device="cuda", dtype=torch.int32)])
    e = torch.zeros(4, dtype=torch.int32, device="cuda")
    o, _ = x.run(x.state, err=e)
    assert e[0] == 0 and torch.isfinite(o).all()


# ---------------- streams, graphs, repeats ----------------

@pytest.mark.parametrize("lens", [[3, 1], [100, 70]])
def test_another_stream_and_a_replayed_graph(lens):
    x = Tokens(lens, seed=9)
    ref_s = x.state.clone()
    refs = [x.run(ref_s)[0].clone() for _ in range(3)]
    s = x.state.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    outs = [x.run(s, stream=stream)[0] for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, refs)) and torch.equal(s, ref_s)
    s, ws = x.state.clone(), kx.gated_delta_workspace(x.q, x.v, x.starts, x.max_len)
    out = torch.empty_like(refs[0])
    x.run(s.clone(), out=out, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.run(s, out=out, ws=ws)
    for r in refs:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r)
        x.run(x.state.clone(), ws=ws)  # eager work between the replays, on the same workspace
    assert torch.equal(s, ref_s)


def test_verify_and_commit_in_a_graph():
    x = Tokens([6, 20], seed=10)
    mask = kx.tree_mask([list(range(-1, 5)), list(range(-1, 19))]).cuda()
    count = i32([3, 9])

    def one(state, o=None, u=None, g=None):
        o, u, g, _ = x.verify(state, mask, out=o, u=u, decay=g)
        kx.gated_delta_commit(x.k, u, g, state, x.starts, count, max_count=20, slots=x.slots)
        return o, u, g
    want = x.state.clone()
    bufs = [t.clone() for t in one(want)]
    refs = [bufs[0].clone()] + [one(want)[0].clone() for _ in range(2)]
    s = x.state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(s, *bufs)
    for r in refs:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bufs[0], r)
    assert torch.equal(s, want)


def test_python_refusals():
    x = Tokens([4, 3], seed=11)
    mask = torch.ones(7, 1, dtype=torch.int64, device="cuda")

    def no(text, f, **change):
        old = {k: getattr(x, k) for k in change}
        for k, v in change.items():
            setattr(x, k, v)
        with pytest.raises(SxError, match=text):
            f()
        for k, v in old.items():
            setattr(x, k, v)
    run, ver = lambda: x.run(x.state), lambda: x.verify(x.state, mask)
    for f in (run, ver):
        no("q must be BF16", f, q=x.q.float())
        no("tokens, heads, dim", f, q=x.q[0])
        no("dense rows", f, v=x.v.transpose(0, 2).contiguous().transpose(0, 2))
        no("a must be", f, a=x.a[:, :2])
        no("slots must be", f, slots=x.slots.long())
        no("A_log must be", f, A_log=x.A_log.double())
        no("on cpu", f, starts=x.starts.cpu())
        no("heads = ", f, q=x.q[:, :1].expand(-1, 3, -1), k=x.k[:, :1].expand(-1, 3, -1))
    with pytest.raises(SxError, match="state must be"):
        x.run(x.state.transpose(2, 3))
    with pytest.raises(SxError, match="mask must be"):
        x.verify(x.state, mask.int())
    with pytest.raises(SxError, match="max_new"):
        kx.gated_delta_verify(x.q, x.k, x.v, x.a, x.b, x.state, x.starts, mask, 65, **x.kw())
    with pytest.raises(SxError, match="overlaps"):
        x.run(x.state, out=x.v)
    with pytest.raises(SxError, match="workspace"):
        x.run(x.state, max_len=40, ws=torch.empty(4, dtype=torch.int64, device="cuda"))
