"""The gated delta rule on cuda:0 where its sums cancel, where starts fall, where a gate forgets everything and where a key has no
length: the three forms (steps, prompts in chunks, drafted trees with their commit) give one answer.

Tolerances as in test_gpu_delta.py (u16 = 2^-8, u32 = 2^-24; c roundings a step)."""
import math

import pytest
import torch

from strixite_amd import kernels as kx
from tests.test_gpu_delta import BF, U16, U32, Tokens, close, gen, i32

pytestmark = pytest.mark.gpu


def chains(lens):
    return [list(range(-1, n - 1)) for n in lens]


def through(x, form):
    """out and the states behind the tokens, by one of the forms."""
    got = x.state.clone()
    if form == "verify":
        out, u, decay, _ = x.verify(got, kx.tree_mask(chains(x.lens)).cuda())
        kx.gated_delta_commit(x.k, u, decay, got, x.starts, i32(x.lens), max_count=max(x.lens), slots=x.slots)
    else:
        out, _ = x.run(got, max_len=16 if form == "steps" else max(64, x.max_len))
    return out, got


# ---------------- sums that cancel ----------------

@pytest.mark.parametrize("Dk,Dv,n,form", [(128, 128, 16, "steps"), (128, 128, 40, "prompt"), (128, 64, 150, "prompt"), (64, 64, 64, "prompt"),
                                          (128, 128, 6, "verify"), (128, 64, 24, "verify"), (64, 128, 64, "verify")])
def test_an_overwritten_value_leaves_nothing_of_itself(Dk, Dv, n, form):
    """The state holds one key's value of 2^12; the first token writes zero there (beta 1, no decay), the others' keys and values are
    small change, and every query is that key. An output is the state's large share less the first token's, both FP32: each is a
    sum of at most 128 products and a few factors, 2-norm 16 u32 of scale |value| the two together less than 32 (sums of 128
    products 6 u32 of their norm, factors and their products under 8)."""
    x = Tokens([n], Hk=2, Hv=4, Dk=Dk, Dv=Dv, raw=True, f32=True, slots=False, seed=Dk + n)
    x.a.zero_(), x.b.fill_(1.0)
    x.v.mul_(2.0 ** -6)
    x.v[0] = 0
    x.q[:] = x.k[:1]
    k0 = x.k[0].double()
    k0 = (k0 / (k0.pow(2).sum(1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(2, 0)
    value = 4096 * torch.randn(4, Dv, device="cuda", generator=gen(n)).double()
    x.state = (k0[:, :, None] * value[:, None, :]).float()[None].contiguous()
    ref, states, _, _, _, _ = x.rule(parents=chains([n]) if form == "verify" else None)
    out, got = through(x, form)
    big = Dk ** -0.5 * value.norm(dim=1)
    d = (out.double() - ref).norm(dim=2)
    print(form, "worst / u32 of the value:", float(((d - U16 * ref.norm(dim=2)).clamp(min=0) / big).max() / U32))
    assert (d <= U16 * ref.norm(dim=2) + 32 * U32 * big).all()


# ---------------- starts that fall ----------------

def possible(starts, T, most):
    """The sequences that the contract serves: possible words, and no start before them that falls."""
    ok, rises = [], True
    for t0, t1 in zip(starts, starts[1:]):
        rises = rises and t1 >= t0
        ok.append(rises and t0 >= 0 and t1 <= T and t1 - t0 <= most)
    return ok


@pytest.mark.parametrize("form", ["steps", "prompt", "verify"])
@pytest.mark.parametrize("starts", [[200, 400, 0, 200], [0, 300, 50, 350], [0, 60, 40, 100], [0, 5, 3, 8], [10, 0, 16], [0, 64, 64, 63, 127, 140], [50, 60, 20, 80, 90],
                                    [-7, 9, 20, 15, 30], [0, 9, 2 ** 31 - 1, 20, 40], [0, 12, -2 ** 31, 12, 25]])
def test_sequences_from_a_falling_start_on_are_left_alone(starts, form):
    B, T = len(starts) - 1, 400
    limit = {"steps": 16, "prompt": 400, "verify": 64}[form]
    x = Tokens([T] + [0] * (B - 1), Hk=1, Hv=2, Dk=64, Dv=64, seed=B)
    ok, at = possible(starts, T, limit), i32(starts)
    mask = (2 ** 63 - 1) * torch.ones(T, 1, dtype=torch.int64, device="cuda")  # every token before its own: a chain

    def call(starts, state, out, err):
        if form != "verify":
            return kx.gated_delta(x.q, x.k, x.v, x.a, x.b, state, starts, limit, **x.kw(out=out, err=err))
        _, u, decay, _ = kx.gated_delta_verify(x.q, x.k, x.v, x.a, x.b, state, starts, mask, limit, **x.kw(out=out, err=err))
        n = starts[1:] - starts[:-1]
        kx.gated_delta_commit(x.k, u, decay, state, starts, torch.where((n > 0) & (n <= limit), n, 0).to(torch.int32), max_count=limit, slots=x.slots)
    for again in range(3):
        state, out, err = x.state.clone(), torch.full((T, 2, 64), 7.0, dtype=BF, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
        call(at, state, out, err)
        want, want_out = x.state.clone(), torch.full_like(out, 7.0)
        for b in range(B):
            if ok[b]:  # alone, its words where they were
                lone = [starts[b]] * (b + 1) + [starts[b + 1]] * (B - b)
                call(i32(lone), want, want_out, None)
        assert torch.equal(out, want_out) and torch.equal(state, want)
        word = err.tolist()
        assert word[0] == (not all(ok)) and (all(ok) or (not ok[word[2]] and word[1] == starts[word[2]]))


def test_many_sequences_with_one_falling_start():
    B, n = 1000, 20
    x = Tokens([n] * B, Hk=1, Hv=1, Dk=64, Dv=16, seed=1)
    clean = x.state.clone()
    ref, _ = x.run(clean)
    for at in (1, 255, 256, 700, 999):
        starts = x.starts.clone()
        starts[at] = starts[at - 1] - 1
        state, out = x.state.clone(), torch.full_like(ref, 7.0)
        kx.gated_delta(x.q, x.k, x.v, x.a, x.b, state, starts, n + 1, **x.kw(out=out))
        assert torch.equal(out[:(at - 1) * n], ref[:(at - 1) * n]) and (out[(at - 1) * n:] == 7).all()
        served = [x.slot(b) for b in range(at - 1)]
        rest = [i for i in range(state.shape[0]) if i not in set(served)]
        assert torch.equal(state[served], clean[served]) and torch.equal(state[rest], x.state[rest])


# ---------------- gates that forget everything ----------------

class Resets(Tokens):
    def gates(self):
        g, beta = super().gates()
        return g.clamp(min=-100.0), beta  # e^-100 of a state is nothing beside u32 |v|, and the tolerance stays a number


@pytest.mark.parametrize("form,lens", [("steps", [16, 9]), ("prompt", [40, 90, 6]), ("prompt", [16, 9]), ("verify", [24, 9]), ("verify", [64, 6])])
@pytest.mark.parametrize("how", ["-inf", "-1e4", "-3e38", "a = inf", "overflow"])
def test_full_resets(form, lens, how):
    x = Resets(lens, Hk=2, Hv=4, raw=how[0] == "-", f32=how != "a = inf", seed=len(lens) + lens[0])
    at = [0, 3, 7, lens[0] - 1, lens[0] + 5]
    if how == "overflow":  # exp(A_log) softplus is past FP32's largest
        x.A_log[1] = 88.0
        x.dt_bias[:] = 0.0
        x.a[:, 1] = 0.5 * x.a[:, 1].abs()  # every token of this head
        for t in at:
            x.a[t, 1] = 1000.0
    else:
        for t in at:
            x.a[t, 1:3] = math.inf if how == "a = inf" else float(how)
    ref, states, _, _, tol, stol = x.rule(parents=chains(lens) if form == "verify" else None, chunked=form != "steps")
    out, got = through(x, form)
    close(out, ref, tol, U16, "out")
    for b, n in enumerate(lens):
        want, e = x.nodes[b][-1]
        mine = got[x.slot(b)]
        assert torch.isfinite(mine).all() and (mine.double() - want).norm() <= 40 * U32 * want.norm(), b


@pytest.mark.parametrize("Dk", [64, 128])
def test_a_reset_is_the_same_token_in_every_form(Dk):
    """A token that forgets everything and one behind it: the three forms' outputs and states, against each other."""
    x = Tokens([12, 3], Hk=1, Hv=2, Dk=Dk, Dv=64, seed=Dk)
    x.a[5, 0] = math.inf
    x.a[13] = math.inf
    (o1, s1), (o2, s2), (o3, s3) = (through(x, f) for f in ("steps", "prompt", "verify"))
    for o, s in ((o2, s2), (o3, s3)):
        assert torch.isfinite(o).all() and torch.isfinite(s).all()
        assert (o.double() - o1.double()).norm() <= 2 * U16 * o1.double().norm() and (s.double() - s1.double()).norm() <= 40 * U32 * s1.double().norm()
    # what came before the reset is gone: a state of other numbers ends as this one does
    y = x.state.clone()
    x.state = torch.where(torch.arange(x.state.shape[0], device="cuda")[:, None, None, None] == x.slot(1), -3 * y, y)
    for f, s in zip(("steps", "prompt", "verify"), (s1, s2, s3)):
        assert torch.equal(through(x, f)[1][x.slot(1)], s[x.slot(1)]), f


# ---------------- keys and queries without a length ----------------

@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("form,n,at", [("steps", 9, 4), ("prompt", 9, 4), ("prompt", 100, 70), ("verify", 9, 4), ("verify", 40, 33)])
def test_a_key_whose_squares_overflow_is_no_number(form, n, at, normalize):
    x = Tokens([n, 2], Hk=2, Hv=4, seed=n + at, normalize=normalize, raw=not normalize)
    ref, refs = through(x, form)
    x.k[at, 0, 3] = 2.0 ** 65
    out, got = through(x, form)
    assert torch.equal(out[n:], ref[n:]) and torch.equal(out[:, 2:], ref[:, 2:]) and torch.equal(got[:, 2:], refs[:, 2:])
    assert out[at:n, :2].isnan().all() and got[x.slot(0), :2].isnan().all() and torch.equal(got[x.slot(1)], refs[x.slot(1)])
    before, was = out[:at].double(), ref[:at].double()  # (verify: products of tokens in FP32 where one is no number)
    assert torch.equal(before, was) if form != "verify" else (before - was).norm() <= 2 * U16 * was.norm()


@pytest.mark.parametrize("form,n,at", [("steps", 9, 4), ("prompt", 100, 70), ("verify", 40, 33)])
def test_a_query_whose_squares_overflow_is_its_own_rows_loss(form, n, at):
    x = Tokens([n, 2], Hk=2, Hv=4, seed=n + at)
    ref, refs = through(x, form)
    x.q[at, 0, 3] = 2.0 ** 65
    out, got = through(x, form)
    assert out[at, :2].isnan().all() and torch.equal(got, refs) and torch.equal(out[at, 2:], ref[at, 2:])
    rest = [i for i in range(n + 2) if i != at]
    assert torch.equal(out[rest], ref[rest])


# ---------------- sums that overflow ----------------

@pytest.mark.parametrize("form,n,at", [("steps", 12, 5), ("prompt", 12, 5), ("prompt", 100, 40), ("prompt", 100, 70), ("verify", 12, 5), ("verify", 50, 20)])
def test_a_correction_too_large_for_fp32_reaches_only_what_is_behind_it(form, n, at):
    """A value of 3e38 under the key that the token before gave -3e38: the correction is not in FP32's range. Rows before it, other
    columns, heads and sequences are as they are without the second value."""
    x = Tokens([n, 3], Hk=1, Hv=2, Dk=64, Dv=64, raw=True, f32=True, seed=n + at)
    x.a.zero_(), x.b.fill_(1.0)
    x.k[at] = x.k[at - 1]
    ref, refs = through(x, form)
    x.v[at - 1, 0, 7], x.v[at, 0, 7] = -3e38, 3e38
    out, got = through(x, form)
    near = lambda a, b: torch.equal(a, b) or form == "verify" and (a.double() - b.double()).norm() <= 2 * U16 * b.double().norm()  # products of tokens in FP32 there
    assert near(out[:at - 1, 0, 7], ref[:at - 1, 0, 7]) and torch.isfinite(out[at - 1, 0, 7])
    assert not torch.isfinite(out[at:n, 0, 7]).any() and not torch.isfinite(got[x.slot(0), 0, :, 7]).any()
    for o, r in ((out[:, 0, :7], ref[:, 0, :7]), (out[:, 0, 8:], ref[:, 0, 8:]), (out[:, 1], ref[:, 1]), (out[n:], ref[n:])):
        assert near(o, r)
    assert torch.equal(got[x.slot(1)], refs[x.slot(1)]) and torch.equal(got[x.slot(0), 1], refs[x.slot(0), 1])
