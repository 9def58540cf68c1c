"""The gated delta rule on cuda:0 where its sums cancel, in its three forms: steps, prompts in chunks, drafted trees with their commit.

Tolerances as in test_gpu_delta.py (u16 = 2^-8, u32 = 2^-24; c roundings a step)."""
import pytest
import torch

from strixite_amd import kernels as kx
from tests.test_gpu_delta import BF, U16, U32, Tokens, gen, i32

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
