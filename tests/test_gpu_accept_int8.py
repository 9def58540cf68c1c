"""Acceptance by the target's probabilities, the 8-bit integer linear and the norms around a block on cuda:0 against plain
implementations in 64 bits.

Whole numbers (tokens, counts, codes) have to be equal. linear: the sum of the codes is exact, then three FP32 roundings, 3 u32 |y|,
and a BF16 store's u16 |y| (u16 = 2^-8, half a step; u32 = 2^-24). norm: y and residual one rounding of an FP64 value, through FP32 for
BF16 (u16 + u32), scale u32.
"""
import math

import pytest
import torch

from strixite_amd import ACT_BF16, ACT_F32, SxError
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


# ---------------- 8-bit integer linear ----------------

def codes(M, K, seed):
    return torch.randint(-128, 128, (M, K), device="cuda", generator=gen(seed), dtype=torch.int8)


@pytest.mark.parametrize("out", [ACT_BF16, ACT_F32])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 4096, 4096), (6, 300, 112), (16, 17, 128), (17, 160, 2560), (33, 1000, 144), (64, 4096, 1040), (48, 9000, 256),
    (65, 131, 272), (100, 5000, 2048), (257, 777, 1600), (300, 12288, 512), (700, 2560, 4096), (1531, 1300, 48), (1000, 4104, 640),
])
def test_linear_int8(M, N, K, out):
    x, w = codes(M, K, M), codes(N, K, N)
    xs, ws = torch.rand(M, device="cuda", generator=gen(1)) + 0.01, torch.rand(N, device="cuda", generator=gen(2)) * 0.02
    xs[M // 2] = 0.0
    y = kx.linear_int8(x, xs, kx.Int8Weight(w, ws), out_act=out)
    ref = torch.cat([(x.double() @ w[r:r + 2048].double().T) for r in range(0, N, 2048)], dim=1) * xs.double()[:, None] * ws.double()
    assert (y.double() - ref).abs().le((3 * U32 + (U16 if out == ACT_BF16 else 0)) * ref.abs() + 1e-38).all()


def test_linear_int8_at_the_ends():
    """The largest sums that 32 bits hold, and sums that cancel to a few units."""
    K = 131056
    x, w = torch.full((70, K), -128, dtype=torch.int8, device="cuda"), torch.full((130, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, ::2], w[2, 1::2], w[2, 0] = -128, 127, 127
    one = torch.ones(130, device="cuda")
    for M in (3, 70):
        y = kx.linear_int8(x[:M], one[:M], kx.Int8Weight(w, one), out_act=ACT_F32)
        want = torch.tensor([16384 * K, -16256 * K, 64 * K - 128 * 255], dtype=torch.float64).float().cuda()
        assert torch.equal(y[:, :3], want.expand(M, 3)) and torch.equal(y[:, 3], y[:, 0])


def test_linear_int8_odd_places_streams_and_graphs():
    x, w = codes(100, 512, 1), codes(77, 512, 2)
    xs, ws = torch.rand(100, device="cuda"), torch.rand(77, device="cuda")
    weight = kx.Int8Weight(w, ws)
    ref = kx.linear_int8(x, xs, weight)
    buf = torch.full((100 * 77 + 3,), 5.0, dtype=BF, device="cuda")
    y = buf[1:1 + 7700].view(100, 77)
    kx.linear_int8(x, xs, weight, y=y)
    assert torch.equal(y, ref) and buf[0] == 5 and (buf[7701:] == 5).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = kx.linear_int8(x, xs, weight, stream=s)
    s.synchronize()
    assert torch.equal(y, ref)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(ref)
    with torch.cuda.graph(graph):
        kx.linear_int8(x, xs, weight, y=out)
    for i in range(3):
        x.copy_(codes(100, 512, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kx.linear_int8(x, xs, weight))


def test_linear_int8_refusals():
    x, w, s = codes(4, 64, 1), codes(8, 64, 2), torch.ones(8, device="cuda")
    weight = kx.Int8Weight(w, s)
    for f, text in [(lambda: kx.Int8Weight(w[:, :24], s), "multiple of 16"), (lambda: kx.Int8Weight(w, s[:4]), "scale must be"),
                    (lambda: kx.Int8Weight(w.float(), s), "q must be"), (lambda: kx.linear_int8(x[:, :32], s[:4], weight), "x must be"),
                    (lambda: kx.linear_int8(x, s, weight), "x_scale must be"), (lambda: kx.linear_int8(x, s[:4], weight, out_act=3), "dtype"),
                    (lambda: kx.linear_int8(x, s[:4].cpu(), weight), "on cpu")]:
        with pytest.raises(SxError, match=text):
            f()


# ---------------- norms around a block ----------------

ACTS = {"none": lambda z: z, "silu": lambda z: z / (1 + torch.exp(-z)), "sigmoid": lambda z: 1 / (1 + torch.exp(-z))}


def norm_reference(x, post, gate, residual, pre, group, act, rs, bs, w_add, eps):
    M, K = x.shape
    h = x.double()
    if post is not None:
        h = h.view(M, -1, group or K)
        h = (h / torch.sqrt(h.square().mean(2, keepdim=True) + eps)).flatten(1) * (post.double().repeat(K // post.numel()) + w_add)
    if gate is not None:
        h = h * ACTS[act](gate.double())
    r = bs * h
    res = None
    if residual is not None:
        res = (rs * residual.double() + r).to(x.dtype)
        r = res.double()
    t = y = r
    if pre is not None:
        t = r * (pre.double() + w_add)
        y = t / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    top = t.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(t * 127.0 / top), torch.zeros_like(t)).to(torch.int8)
    return y, q, (y.abs().amax(1) / 127.0), res


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M,K,group,parts,act", [
    (1, 8, None, "PGRp", "none"), (6, 4096, None, "PGRp", "none"), (5, 2560, 128, "PG", "silu"), (3, 16384, 64, "PGR", "sigmoid"), (9, 4096, 512, "Pp", "none"),
    (7, 512, 8, "PGR", "silu"), (33, 520, None, "PRp", "none"), (200, 1024, None, "Rp", "none"), (2, 1288, None, "p", "none"), (4, 2048, None, "G", "sigmoid"),
    (257, 136, None, "R", "none"), (3, 9000, None, "PG", "silu"), (65, 256, 128, "sPGR", "silu"), (4, 640, None, "", "none"), (2, 8200, None, "PGRp", "silu"),
])
def test_block_norm(M, K, group, parts, act, dtype):
    g = gen(M + K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    wide = r(M, K + 16)
    x = wide[:, :K]
    post = (r(group if "s" in parts else K) * 0.3).to(dtype) if "P" in parts else None
    gate = r(M, K) if "G" in parts else None
    residual = r(M, K) * 3 if "R" in parts else None
    pre = (r(K) * 0.3).to(dtype) if "p" in parts else None
    if M > 2:
        x[1] = 0  # a row of zeros
        if residual is not None:
            residual[1] = 0
    y = torch.empty(M, K, dtype=dtype, device="cuda")
    # scales and shifts that 32 bits hold exactly
    kw = dict(group=group, gate_act=act, residual_scale=0.75, branch_scale=1.25, w_add=1.0, eps=2.0 ** -20)
    q, s, res = kx.block_norm_int8(x, post, gate, residual, pre, y=y, **kw)
    ry, rq, rs, rres = norm_reference(x, post, gate, residual, pre, group, act, 0.75, 1.25, 1.0, 2.0 ** -20)
    assert torch.equal(q, rq)
    assert (res is None) == (rres is None) and (res is None or torch.equal(res, rres))
    assert (s.double() - rs).abs().le(1.01 * U32 * rs).all()
    assert (y.double() - ry).abs().le((U32 * 1.01 if dtype != BF else U16 + 2 * U32) * ry.abs() + 1e-38).all()
    if M > 2:
        assert s[1] == 0 and (q[1] == 0).all()


def test_block_norm_one_gate_for_all_rows_and_in_place():
    g = gen(3)
    x, res = torch.randn(20, 256, device="cuda", generator=g).to(BF), torch.randn(20, 256, device="cuda", generator=g).to(BF)
    gate, post = torch.randn(256, device="cuda", generator=g).to(BF), torch.randn(256, device="cuda", generator=g).to(BF)
    a = kx.block_norm_int8(x, post, gate[None].expand(20, 256), res, None)
    b = kx.block_norm_int8(x, post, gate[None].expand(20, 256).contiguous(), res, None)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    keep = res.clone()
    c = kx.block_norm_int8(x, post, gate[None].expand(20, 256), keep, None, residual_out=keep, y=x)
    assert c[2] is keep and torch.equal(keep, a[2]) and torch.equal(c[0], a[0]) and torch.equal(x, keep)
    q, s, r = kx.block_norm_int8(x, post, None, res, None, codes=False)
    assert q is None and s is None and r is not None


def test_block_norm_ties_and_rows_without_a_scale():
    # 127 t / amax is k + 1/2 for t = (2 k + 1) amax / 254: amax 254 and whole numbers
    x = torch.zeros(4, 256, device="cuda")
    x[0, 0], x[0, 1:127] = 254.0, torch.arange(1, 127, device="cuda").float() * 2 - 1
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    q, s, _ = kx.block_norm_int8(x)
    assert torch.equal(q[0, 1:127].double(), torch.round(x[0, 1:127].double() / 2)) and q[0, 0] == 127 and s[0] == 2
    assert s[1].isnan() and s[2].isnan() and (q[1:] == 0).all() and s[3] == 0
    y = torch.empty_like(x)
    kx.block_norm_int8(x, post=torch.ones(256, device="cuda"), y=y)
    assert y[1].isnan().all() and torch.isfinite(y[0]).all() and (y[3] == 0).all()


def test_block_norm_ties_are_those_of_the_formula_in_64_bits():
    """Few distinct values and no residual between the norm and the codes, so that products stand on a border between two codes:
    the rounding of x / root says which. The squares' sum is exact in 64 bits, so every order of adding gives the same root (the mean is
    the sum times the rounded 1 / K)."""
    for M, K, group, gated, pre, seed in [(512, 4096, 0, False, False, 1), (512, 1024, 0, False, True, 2), (256, 1024, 0, True, False, 3),
                                          (256, 2048, 64, False, False, 4), (256, 512, 512, True, True, 5), (512, 2560, 0, False, False, 6)]:
        g = gen(seed)
        draw = lambda *shape: (torch.randint(-12, 13, shape, generator=g, device="cuda").float() / 8).bfloat16()
        x, post = draw(M, K), draw(K) + 2
        gate, w = draw(M, K) if gated else None, draw(K) + 2 if pre else None
        q, _, _ = kx.block_norm_int8(x, post, gate, None, w, eps=1e-6, group=group or None, gate_act="none")
        h = x.double().cpu().view(M, -1, group or K)
        mean = h.square().sum(2, keepdim=True) * (1.0 / (group or K)) + 1e-6
        root = torch.tensor([math.sqrt(v) for v in mean.flatten().tolist()], dtype=torch.float64).view(mean.shape)  # the nearest; torch's here is not always
        h = (h / root).flatten(1) * post.double().cpu()
        h = h * gate.double().cpu() if gated else h
        h = h * w.double().cpu() if pre else h
        n = h * 127.0 / h.abs().amax(1, keepdim=True)
        assert ((n - n.floor() - 0.5).abs() < 1e-12).any(), "no product near a border"
        assert torch.equal(q.cpu(), torch.round(n).to(torch.int8)), (M, K, group, gated, pre)


def test_block_norm_streams_and_graphs():
    g = gen(4)
    x, w = torch.randn(40, 2560, device="cuda", generator=g).to(BF), torch.randn(2560, device="cuda", generator=g).to(BF)
    ref = kx.block_norm_int8(x, post=w, residual=x.flip(0), pre=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    res = x.flip(0)
    torch.cuda.synchronize()
    got = kx.block_norm_int8(x, post=w, residual=res, pre=w, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    q, sc, out = (torch.empty_like(t) for t in ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kx.block_norm_int8(x, post=w, residual=res, pre=w, q=q, scale=sc, residual_out=out)
    for _ in range(3):
        q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, ref[0]) and torch.equal(sc, ref[1]) and torch.equal(out, ref[2])


def test_block_norm_refusals():
    x, w = torch.ones(4, 256, device="cuda", dtype=BF), torch.ones(256, device="cuda", dtype=BF)
    for kw, text in [(dict(post=w.float()), "post must be"), (dict(post=w[:64], group=128), "post must be"), (dict(post=w, group=96), "group = 96"),
                     (dict(post=w, group=1024), "group = 1024"), (dict(gate=w), "gate must be"), (dict(gate_act="gelu"), "gate_act"), (dict(pre=w[:8]), "pre must be"),
                     (dict(residual=x[:2]), "residual must be"), (dict(residual_out=x), "without a residual"), (dict(y=x[:, :8]), "y must be"),
                     (dict(eps=-1.0), "eps"), (dict(branch_scale=math.inf), "branch_scale"), (dict(codes=False), "no output"),
                     (dict(codes=False, q=torch.empty(4, 256, dtype=torch.int8, device="cuda")), "without codes"), (dict(pre=w.cpu()), "on cpu")]:
        with pytest.raises(SxError, match=text):
            kx.block_norm_int8(x, **kw)
    with pytest.raises(SxError, match="multiple of 8"):
        kx.block_norm_int8(x[:, :20])
    buf = torch.ones(5, 256, device="cuda", dtype=BF)
    with pytest.raises(SxError, match="overlaps an input at other rows"):
        kx.block_norm_int8(buf[:4], y=buf[1:])
    with pytest.raises(SxError, match="overlap"):
        kx.block_norm_int8(x, residual=buf[:4], residual_out=buf[:4], y=buf[1:])


# ---------------- acceptance ----------------

def accept_reference(logits, drafts, starts, u, temperature, n, draft_logits=None, V=None):
    """Row by row on the host; a row's tokens in order. Also the least distance of a draw to a border, for the test's own check."""
    V = logits.shape[1] if V is None else V
    L, D = logits[:, :V].double().cpu(), None if draft_logits is None else draft_logits.double().cpu()
    drafts, starts, u, temperature = drafts.tolist(), starts.tolist(), u.cpu(), temperature.tolist()
    B = len(starts) - 1
    tokens, count, status = torch.full((B, n), -1, dtype=torch.int32), [], []
    for b in range(B):
        t, end, j, st = starts[b], starts[b + 1], 0, 0
        if t == end:
            count.append(0), status.append(0)
            continue
        while True:
            row, last, d = L[t + j], t + j + 1 == end, drafts[t + j]
            T = temperature[b]
            bad = bool(row.isnan().any()) or not math.isfinite(float(row.max())) or not math.isfinite(T)
            if not last and not 0 <= d < V:
                bad = True
            if not bad and not last and T > 0 and D is not None:
                bad = bool(D[t + j].isnan().any()) or not math.isfinite(float(D[t + j].max()))
            if bad:
                st = 1 + j
                break
            if T <= 0:
                tok = int((row == row.max()).nonzero()[0])
                if not last and tok == d:
                    tokens[b, j] = d
                    j += 1
                    continue
                tokens[b, j] = tok
                break
            p = torch.exp((row - row.max()) / T)
            p /= p.sum()
            w = p
            if not last:
                q = torch.zeros(V, dtype=torch.float64)
                if D is None:
                    q[d] = 1.0
                else:
                    e = torch.exp((D[t + j] - D[t + j].max()) / T)
                    q[:D.shape[1]] = e / e.sum()
                if float(u[t + j, 0]) * float(q[d]) < float(p[d]):
                    tokens[b, j] = d
                    j += 1
                    continue
                w = (p - q).clamp(min=0)
                if float(w.sum()) == 0:
                    w = p
            c = w.cumsum(0)
            tokens[b, j] = int(torch.searchsorted(c, u[t + j, 1] * c[-1], right=True).clamp(max=int(w.nonzero()[-1])))
            break
        count.append(j if st else j + 1), status.append(st)
    return tokens, torch.tensor(count, dtype=torch.int32), torch.tensor(status, dtype=torch.int32)


class Drafts:
    def __init__(self, lens, V, Vd=0, dtype=torch.float32, seed=0, temps=None, near=0.5, ld=0):
        g = gen(seed)
        T = sum(lens)
        self.n, self.starts = max(lens + [1]), i32([0] + torch.tensor(lens).cumsum(0).tolist())
        wide = (2.5 * torch.randn(T, V + ld, device="cuda", generator=g)).to(dtype)
        self.logits = wide[:, :V]
        self.draft_logits = (self.logits[:, :Vd].float() + near * torch.randn(T, Vd, device="cuda", generator=g)).to(dtype) if Vd else None
        guess = (self.logits if not Vd else self.draft_logits).float()
        noise = -torch.log(-torch.log(torch.rand(guess.shape, device="cuda", generator=g).clamp(1e-20, 1 - 1e-7)))
        self.drafts = (guess + (noise if Vd else 0.2 * noise)).argmax(1).to(torch.int32)
        self.u = torch.rand(T, 2, dtype=torch.float64, device="cuda", generator=g)
        B = len(lens)
        self.temperature = torch.tensor(temps if temps else [0.8] * B, device="cuda")

    def run(self, **kw):
        return kx.mtp_accept_sampled(self.logits, self.drafts, self.starts, self.u, self.temperature, self.n, **{**dict(draft_logits=self.draft_logits), **kw})

    def check(self, **kw):
        got = self.run(**kw)
        want = accept_reference(self.logits, self.drafts, self.starts, self.u, self.temperature, self.n, self.draft_logits, kw.get("n_valid"))
        for a, b, what in zip(got, want, ("tokens", "count", "status")):
            assert torch.equal(a.cpu(), b), (what, a.tolist(), b.tolist())
        return got


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("lens,V,Vd", [
    ([1], 7, 0), ([1, 1], 2048, 2048), ([6], 5000, 0), ([6], 5000, 5000), ([4, 0, 1, 9], 2049, 1500), ([16] * 12, 4097, 4097), ([3, 5], 151936, 120000),
    ([2] * 40, 600, 600), ([6, 2], 248320, 0), ([64, 3], 300, 200), ([256], 50, 50), ([5, 5, 5], 1, 1),
])
def test_accept(lens, V, Vd, dtype):
    for seed in range(3):
        Drafts(lens, V, Vd, dtype, seed).check()


def test_accept_mixed_temperatures_and_wide_rows():
    for Vd in (0, 3000):
        x = Drafts([6, 6, 6, 1, 6, 3], 4000, Vd, seed=5, temps=[0.0, 1.0, 1e-3, 0.0, 100.0, -1.0], near=0.2, ld=37)
        x.drafts[:4] = x.logits[:4].argmax(1).to(torch.int32)
        got = x.check()
        assert int(got[1][0]) >= 5
        x.check(n_valid=3500) if Vd else x.check(n_valid=int(x.drafts.max()) + 1)


def test_accept_greedy_ties_take_the_lowest_place():
    x = Drafts([2, 1], 5000, seed=1, temps=[0.0, 0.0])
    x.logits[:] = -1.0
    x.logits[0, 4000] = x.logits[0, 77] = 3.0
    x.logits[1, 4999] = x.logits[1, 2048] = 2.0
    x.drafts[0] = 77
    tokens, count, _ = x.check()
    assert tokens[0].tolist() == [77, 2048] and count.tolist() == [2, 1] and tokens[1].tolist() == [0, -1]


def test_accept_masked_vocabularies_and_certain_rows():
    """-inf logits have no probability in either; a row with one token left; draws at 0 and just under 1."""
    for Vd in (0, 900):
        x = Drafts([3, 3, 3, 3], 1000, Vd, seed=7)
        x.logits[0, 1:] = -math.inf        # p is all on place 0
        x.drafts[0] = 0
        x.logits[3, :990] = -math.inf      # p has nothing where the draft can be
        x.logits[6, ::2] = -math.inf
        x.logits[9, 5:] = -math.inf
        x.u[3:6] = 0.0
        x.u[6:9] = 1 - 2.0 ** -53
        if Vd:
            x.draft_logits[3, 7:] = -math.inf
            x.draft_logits[0, 1:] = -math.inf
            x.drafts[3] = 2
        tokens, _, status = x.check()
        assert tokens[0, 0] == 0 and tokens[1, 0] >= 990 and (status == 0).all()


def test_accept_equal_distributions_keep_every_draft():
    x = Drafts([9], 3000, 3000, seed=2, near=0.0)
    tokens, count, _ = x.check()
    assert count.tolist() == [9] and torch.equal(tokens[0, :8], x.drafts[:8])


def test_accept_rows_without_a_distribution():
    x = Drafts([4] * 7, 3000, 3000, seed=3, near=0.0)
    x.logits[5, 2999] = math.nan       # sequence 1, row 1
    x.logits[8] = -math.inf            # 2, row 0
    x.draft_logits[14, 5] = math.nan   # 3, row 2
    x.draft_logits[15] = math.nan      # 3's last row has no draft
    x.drafts[17] = 3000                # 4, row 1
    x.logits[20, 9] = math.inf         # 5, row 0
    x.temperature[6] = math.nan
    tokens, count, status = x.check()
    assert status.tolist() == [0, 2, 1, 3, 2, 1, 1] and count.tolist() == [4, 1, 0, 2, 1, 0, 0]
    x = Drafts([2, 2], 100, seed=1)
    x.drafts[1], x.drafts[3] = -5, 10 ** 9  # of last rows: nobody's
    x.check()


def test_accept_impossible_starts():
    x = Drafts([4, 4], 500, 500, seed=3)
    ref = x.run()
    for bad in ([0, 9, 8], [0, -1, 8], [0, 4, 9], [0, 4, 2 ** 31 - 1]):
        x.starts = i32(bad)
        tokens, count, status = x.run()
        for b in range(2):
            ok = 0 <= bad[b] <= bad[b + 1] <= 8 and bad[b + 1] - bad[b] <= 4
            assert (int(status[b]) == 0) == ok and (ok or (int(count[b]) == 0 and int(status[b]) == -1 and (tokens[b] == -1).all()))
    assert ref[2].tolist() == [0, 0]


def test_accept_keeps_the_targets_distribution():
    """Over many draws the first token comes out as the target alone would give it (chi-square, 15 degrees, p = 1e-6: 56)."""
    for Vd in (16, 12, 0):
        N = 1024
        x = Drafts([2] * N, 16, Vd, seed=9, temps=[1.0] * N)
        x.logits[:] = x.logits[0]
        counts = torch.zeros(16, dtype=torch.float64)
        for i in range(8):
            g = gen(100 + i)
            if Vd:
                x.draft_logits[:] = x.draft_logits[0]
                x.drafts = torch.multinomial(torch.softmax(x.draft_logits.double(), 1), 1, generator=g)[:, 0].to(torch.int32)
            else:
                x.drafts[:] = 3
            x.u = torch.rand(2 * N, 2, dtype=torch.float64, device="cuda", generator=g)
            counts += torch.bincount(x.run()[0][:, 0].cpu().long(), minlength=16)
        want = torch.softmax(x.logits[0].double().cpu(), 0) * 8 * N
        assert float(((counts - want) ** 2 / want).sum()) < 56


def test_accept_streams_and_graphs():
    x = Drafts([6, 3], 9000, 8000, seed=4)
    ref = x.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = x.run(stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    bufs = dict(zip(("tokens", "count", "status"), (torch.empty_like(t) for t in ref)))
    ws = torch.empty((kx.mtp_accept_sampled_workspace_bytes(9, 2, 9000, 8000) + 7) // 8, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.run(ws=ws, **bufs)
    for i in range(4):
        x.u.copy_(torch.rand(9, 2, dtype=torch.float64, device="cuda", generator=gen(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bufs[k], r) for k, r in zip(bufs, x.run(ws=ws)))


def test_accept_refusals():
    x = Drafts([6, 3], 500, 400, seed=4)
    for kw, text in [(dict(n_valid=501), "n_valid"), (dict(draft_logits=x.draft_logits.to(BF)), "draft_logits must be"), (dict(n_valid=300), "n_draft = 400"),
                     (dict(ws=torch.empty(2, dtype=torch.int64, device="cuda")), "workspace"), (dict(tokens=torch.empty(2, 5, dtype=torch.int32, device="cuda")), "tokens must be"),
                     (dict(draft_logits=x.draft_logits.cpu()), "on cpu")]:
        with pytest.raises(SxError, match=text):
            x.run(**kw)
    with pytest.raises(SxError, match="max_rows"):
        kx.mtp_accept_sampled(x.logits, x.drafts, x.starts, x.u, x.temperature, 257)
    with pytest.raises(SxError, match="u must be"):
        kx.mtp_accept_sampled(x.logits, x.drafts, x.starts, x.u.float(), x.temperature, 6)
