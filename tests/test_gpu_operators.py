"""The attention half of a verify layer and scored routing on cuda:0 against plain implementations in 64 bits.

Tolerances count roundings. u16 = 2^-8 (BF16, half a step), u32 = 2^-24.
  attention: the output's own rounding u16 |o|, and for A = sum_j p_j |v_j| (p the softmax): P's rounding t A (t = 2^-8 with
    one BF16 term, 2^-16 with two, 2^-11 in FP16), the scores' error twice, e = (D + 4) u32 scale sum |q||k| in the
    exponent (numerator and sum), and (keys + 64) u32 A for the FP32 sums and exponentials. FP16 P loses what is under
    2^-25 of the reference maximum: keys 2^-25 max |v| on a sum of at least 2^-8.
  linear: FP32 output (K / 32 + 8) u32 S for S = sum |x||w| with the scales; BF16 output u16 |y| + 2^-12 S (a block's
    largest product keeps 12 bits or more).
  norm: y u16 |y| (FP32: 16 u32 |y|) and (K / 64 + 16) u32 relative for the row's root; scale (K / 64 + 16) u32.
"""
import math

import numpy as np
import pytest
import torch

from strixite_amd import ACT_BF16, ACT_F32
from strixite_amd import kernels as kx

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -8, 2.0 ** -24
F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------- attention ----------------

class Batch:
    """Sequences of cached lengths `lens` and drafted tokens `news`, pages shuffled, a random mask over the drafts."""

    def __init__(self, D, Hq, Hkv, page, lens, news, cache="bf16", seed=0, mask="tree", order="token", spare=0, amp=1.0):
        g, host = gen(seed), torch.Generator().manual_seed(seed)
        self.D, self.Hq, self.Hkv, self.page, self.lens_h, self.news = D, Hq, Hkv, page, lens, news
        B, self.T = len(lens), sum(news)
        self.max_new = max(max(news), 1)
        P = max(1, -(-max(lens) // page))
        pages = B * P + 3
        perm = torch.randperm(pages, generator=host)
        self.table = perm[:B * P].to(torch.int32).view(B, P).cuda()
        rows = self.T + spare
        qkv = (amp * torch.randn(rows, Hq + 2 * Hkv, D, device="cuda", generator=g)).to(BF)
        self.q, self.kn, self.vn = qkv.split([Hq, Hkv, Hkv], dim=1)
        self.ks, self.vs = (0.0625, 0.05) if cache == "fp8" else (1.0, 1.0)

        def filled(sc):
            x = torch.randn(pages, page, Hkv, D, device="cuda", generator=g)
            x = (x / sc).to(F8) if cache == "fp8" else x.to(BF)
            if order == "head":  # [pages, heads, page, dim] in memory
                x = x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
            return x
        self.kc, self.vc = filled(self.ks), filled(self.vs)
        self.lens, self.starts = i32(lens), i32([0] + np.cumsum(news).tolist())
        W = (self.max_new + 63) // 64
        if mask == "tree":
            par = [[-1] + [int(torch.randint(max(-1, i - 5), i, (1,), generator=host)) for i in range(1, n)] if n else [] for n in news]
            m = kx.tree_mask(par)
            m = torch.cat([m, torch.zeros(m.shape[0], W - m.shape[1], dtype=torch.int64)], 1)
        else:  # any subset, some rows see nothing
            m = torch.randint(-2 ** 62, 2 ** 62, (self.T, W), generator=host)
            m[torch.rand(self.T, generator=host) < 0.3] = 0
        self.mask = torch.cat([m, torch.zeros(spare, W, dtype=torch.int64)]).cuda()

    def run(self, **kw):
        return kx.tree_attention(self.q, self.kn, self.vn, self.kc, self.vc, self.table, self.lens, self.starts, self.mask,
                                 self.max_new, k_scale=self.ks, v_scale=self.vs, **kw)

    def terms(self):
        rows = self.max_new * self.Hq // self.Hkv
        two = rows <= 64
        if self.kc.dtype == F8:
            return max(2.0 ** -11, 2.0 ** -16 if two else U16)  # cached FP16, drafted BF16
        return 2.0 ** -16 if two else U16

    def reference(self):
        """out, its tolerance, the log sums and theirs, for every drafted row."""
        G, scale = self.Hq // self.Hkv, self.D ** -0.5
        out = torch.zeros(self.T, self.Hq, self.D, dtype=torch.float64, device="cuda")
        tol, lse, lse_tol = torch.zeros_like(out), torch.zeros(self.T, self.Hq, dtype=torch.float64, device="cuda"), None
        lse_tol = torch.zeros_like(lse)
        t0 = 0
        for b, (L, n) in enumerate(zip(self.lens_h, self.news)):
            if n == 0:
                continue
            ids = self.table[b, :-(-L // self.page)].tolist()
            flat = lambda c, s: (torch.cat([c[i] for i in ids])[:L].double() * s if L else
                                 torch.zeros(0, self.Hkv, self.D, dtype=torch.float64, device="cuda"))
            k = torch.cat([flat(self.kc, self.ks), self.kn[t0:t0 + n].double()])
            v = torch.cat([flat(self.vc, self.vs), self.vn[t0:t0 + n].double()])
            m = self.mask[t0:t0 + n].cpu().tolist()
            see = torch.tensor([[True] * L + [bool(m[i][j >> 6] >> (j & 63) & 1) for j in range(n)] for i in range(n)],
                               device="cuda").repeat_interleave(G, 0)
            for h in range(self.Hkv):
                q = self.q[t0:t0 + n, h * G:(h + 1) * G].double().reshape(n * G, self.D)
                kh, vh = k[:, h].clone(), v[:, h].clone()
                unseen = ~see.any(0)  # a token that no row sees
                kh[unseen], vh[unseen] = 0, 0
                s = (q @ kh.T * scale).masked_fill(~see, -math.inf)
                top = s.amax(1, keepdim=True)
                top = torch.where(top.isinf(), torch.zeros_like(top), top)
                p = torch.exp(s - top)
                l = p.sum(1, keepdim=True)
                p = p / l.clamp(min=1e-300)
                o, A = p @ vh, p @ vh.abs()
                e = ((self.D + 4) * U32 * scale * (q.abs() @ kh.abs().T)).masked_fill(~see, 0).amax(1, keepdim=True)
                keys = L + n
                bound = U16 * o.abs() + (self.terms() + 2 * e + (keys + 64) * U32) * A + keys * 2.0 ** -33 * vh.abs().amax(0)
                shape = (n, G, self.D)
                out[t0:t0 + n, h * G:(h + 1) * G] = o.view(shape)
                tol[t0:t0 + n, h * G:(h + 1) * G] = bound.view(shape)
                lse[t0:t0 + n, h * G:(h + 1) * G] = (top + l.log()).view(n, G)
                lse_tol[t0:t0 + n, h * G:(h + 1) * G] = (e + (keys + 64) * U32 + 4 * U32 * top.abs()).view(n, G)
            t0 += n
        return out, tol, lse, lse_tol


def check(batch, out, lse=None):
    o, tol, l, ltol = batch.reference()
    got = out[:batch.T].double()
    assert torch.isfinite(got).all()
    bad = (got - o).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - o).abs() / tol.clamp(min=1e-300)).max()):.3g} times the tolerance"
    if lse is not None:
        d = lse[:batch.T].double()
        none = l.isinf()
        assert torch.equal(d.isinf(), none)
        assert ((d - l).abs()[~none] <= ltol[~none]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
@pytest.mark.parametrize("Hq,Hkv,page,lens,news,mask,order", [
    (2, 2, 16, [0], [1], "tree", "token"),                       # the first token of all
    (4, 1, 16, [1, 15, 16, 17, 31, 33], [1, 6, 1, 4, 3, 2], "tree", "token"),
    (8, 2, 32, [63, 64, 65, 127, 128, 129], [6, 6, 6, 6, 6, 6], "tree", "head"),
    (4, 2, 64, [0, 300, 1000, 0, 255, 256, 257], [3, 0, 24, 16, 0, 7, 1], "any", "token"),  # rows and sequences with nothing
    (7, 1, 128, [700, 90], [9, 12], "any", "head"),              # 7 heads a key head: ragged row tiles
    (6, 3, 16, [400], [40], "any", "token"),                     # three key heads, 80 rows
    (4, 1, 256, [513, 5], [64, 33], "tree", "token"),            # 256 rows
    (16, 1, 16, [100, 3000], [25, 2], "any", "token"),           # 400 rows: two row groups
    (2, 1, 64, [50, 777], [200, 256], "any", "token"),           # four mask words, 512 rows
])
def test_attention(D, cache, Hq, Hkv, page, lens, news, mask, order):
    print(f"attention D={D} {cache} Hq={Hq} Hkv={Hkv} page={page} lens={lens} news={news}", flush=True)
    b = Batch(D, Hq, Hkv, page, lens, news, cache, seed=D + len(lens), mask=mask, order=order)
    lse = torch.empty(b.T, Hq, device="cuda")
    out, err = b.run(lse=lse, err=torch.zeros(4, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert err.tolist()[0] == 0
    check(b, out, lse)


@pytest.mark.parametrize("Hq,news", [(4, [6]), (4, [12]), (8, [12]), (8, [16]), (8, [24])])
def test_attention_long_and_peaked(Hq, news):
    """Maxima that rise through a long cache (scores of tens), split over every block, each row tile."""
    print(f"attention long Hq={Hq} news={news}", flush=True)
    b = Batch(128, Hq, 1, 64, [9001], news, seed=5, amp=3.0)
    k = b.kc.view(-1, 1, 128)
    b.kc = (k.float() * torch.linspace(0.1, 2.0, k.shape[0], device="cuda").view(-1, 1, 1)).to(BF).view_as(b.kc)
    check(b, b.run()[0])


def test_attention_same_result_twice_and_other_workspace():
    b = Batch(128, 8, 2, 32, [900, 40, 0, 2000], [6, 24, 3, 1], seed=3)
    first = b.run()[0].clone()
    ws = kx.tree_attention_workspace(b.q, b.kn, b.starts, b.max_new)
    ws.fill_(-1)  # nothing in it is read before it is written
    assert torch.equal(b.run(ws=ws)[0], first)
    small = Batch(128, 8, 2, 32, [77], [24], seed=4)
    ref = small.run()[0].clone()
    assert torch.equal(small.run(ws=ws)[0], ref) and torch.equal(b.run(ws=ws)[0], first)


def test_attention_rows_behind_the_last_sequence():
    b = Batch(64, 4, 2, 16, [20, 50], [5, 2], seed=9, spare=4)
    out = torch.full((b.T + 4, 4, 64), 7.0, dtype=BF, device="cuda")
    lse = torch.full((b.T + 4, 4), 7.0, device="cuda")
    b.run(out=out, lse=lse)
    check(b, out, lse)
    assert (out[b.T:] == 7.0).all() and (lse[b.T:] == 7.0).all()


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
@pytest.mark.parametrize("D", [64, 256])
def test_attention_unseen_tokens_and_unused_pages_do_not_matter(D, cache):
    b = Batch(D, 4, 2, 16, [37, 0], [9, 40], cache, seed=13)
    clean = b.run()[0].clone()
    # slots behind a sequence's length, pages of none, and drafted tokens 3 and 20 that few rows see
    for c in (b.kc, b.vc):
        raw = c.view(torch.uint8 if cache == "fp8" else torch.int16)
        used = set(b.table[0, :3].tolist())
        for p in range(c.shape[0]):
            if p not in used:
                raw[p] = 0x7F if cache == "fp8" else 0x7FC0
        raw[int(b.table[0, 2]), 5:] = 0x7F if cache == "fp8" else 0x7F80
    assert torch.equal(b.run()[0], clean)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for which in (b.kn, b.vn):
            keep = which[3].clone()
            which[3] = bad
            got = b.run()[0]
            sees = torch.tensor([bool(w >> 3 & 1) for w in b.mask[:9, 0].tolist()], device="cuda")
            assert torch.equal(got[9:], clean[9:])
            assert torch.equal(got[:9][~sees], clean[:9][~sees])
            if which is b.vn or math.isnan(bad):
                assert not torch.isfinite(got[:9][sees]).all()
            which[3] = keep
    assert torch.equal(b.run()[0], clean)


def test_attention_in_a_graph_with_other_lengths():
    b = Batch(128, 8, 2, 64, [3000, 500], [6, 24], seed=21)
    ws = kx.tree_attention_workspace(b.q, b.kn, b.starts, b.max_new)
    out = torch.empty(b.T, 8, 128, dtype=BF, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.run(ws=ws, out=out)
    for lens in ([3000, 500], [1, 0], [128, 2999], [0, 64], [3000, 3000]):
        b.lens.copy_(i32(lens))
        b.lens_h = lens
        eager = b.run()[0].clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens
        check(b, out)


def test_attention_on_another_stream():
    b = Batch(128, 4, 1, 32, [800], [12], seed=22)
    ref = b.run()[0].clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got, _ = b.run(stream=s)
    s.synchronize()
    assert torch.equal(got, ref)
    with torch.cuda.stream(s):
        got, _ = b.run()
    s.synchronize()
    assert torch.equal(got, ref)


def test_attention_reports_what_it_cannot_read():
    """Lengths past the table, impossible runs and pages outside the cache: NaN rows or none, the other rows as they were,
    the words in err. The kernel looks at each before it makes an address of it."""
    b = Batch(64, 4, 2, 16, [40, 30, 20], [5, 3, 2], seed=31)
    clean = b.run()[0].clone()

    def go(want_err, nan_rows):
        out = torch.zeros(b.T, 4, 64, dtype=BF, device="cuda")
        err = torch.zeros(4, dtype=torch.int32, device="cuda")
        b.run(out=out, err=err)
        torch.cuda.synchronize()
        assert err.tolist()[:3] == want_err
        rows = torch.zeros(b.T, dtype=torch.bool, device="cuda")
        rows[nan_rows] = True
        assert torch.isnan(out[rows].float()).all()
        assert torch.equal(out[~rows], clean[~rows])

    for bad in (49, -1, 2 ** 31 - 1):
        b.lens[1] = bad
        go([1, bad, 1], [5, 6, 7])
    b.lens[1] = 30
    for bad in (-1, b.kc.shape[0], 2 ** 31 - 1):
        keep = int(b.table[0, 1])
        b.table[0, 1] = bad
        go([1, bad, 0], [0, 1, 2, 3, 4])
        b.table[0, 1] = keep
    b.table[2, 2] = -7  # behind sequence 2's length: not looked at
    go([0, 0, 0], [])


def test_attention_past_32_bit_offsets():
    """A cache whose last pages lie more than 2^32 bytes behind its first."""
    D, Hkv, page = 256, 8, 64
    pages = (5 << 30) // (page * Hkv * D * 2)
    kc = torch.empty(pages, page, Hkv, D, dtype=BF, device="cuda")
    vc = torch.empty_like(kc)
    b = Batch(D, 8, Hkv, page, [130], [4], seed=41)
    at = [pages - 1, 3, pages - 2]
    for i, p in enumerate(at):
        kc[p], vc[p] = b.kc[int(b.table[0, i])], b.vc[int(b.table[0, i])]
    b.kc, b.vc, b.table = kc, vc, i32([at])
    check(b, b.run()[0])


# ---------------- cache append ----------------

def e4m3(x):
    """x in 64 bits to the nearest e4m3 value (ties to even), saturating."""
    x = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
@pytest.mark.parametrize("layers,Hkv,D,page,lens,news,count,path", [
    (1, 1, 64, 16, [0], [1], [1], False),
    (3, 2, 128, 16, [15, 16, 0, 33], [4, 6, 1, 3], [4, 2, 0, 3], True),
    (2, 3, 256, 64, [63, 1], [20, 30], [17, 30], True),
    (2, 2, 72, 32, [5, 40], [3, 8], [3, 8], False),     # a head width that attention does not take
])
def test_kv_append(cache, layers, Hkv, D, page, lens, news, count, path):
    print(f"append {cache} layers={layers} D={D} lens={lens}", flush=True)
    if cache == "fp8" and D % 16:
        D += 8  # FP8 strides are multiples of 16 bytes
    g, host = gen(len(lens)), torch.Generator().manual_seed(1)
    B, T = len(lens), sum(news)
    P = -(-(max(lens) + max(news)) // page)
    table = torch.randperm(B * P + 2, generator=host)[:B * P].to(torch.int32).view(B, P).cuda()
    kv = (3 * torch.randn(2, layers, T, Hkv, D, device="cuda", generator=g)).to(BF)
    kv[0, 0, 0, 0, :2] = torch.tensor([1e5, float("nan")], device="cuda")
    shape = (layers, B * P + 2, page, Hkv, D)
    old = torch.randn(2, *shape, device="cuda", generator=g).to(BF if cache == "bf16" else F8)
    ks, vs = (1.0, 1.0) if cache == "bf16" else (0.03, 0.7)
    caches = old.clone()
    p = torch.zeros(B, max(news), dtype=torch.int32)
    for b, n in enumerate(news):
        nodes = torch.randperm(n, generator=host)[:count[b]].sort().values if path else torch.arange(count[b])
        p[b, :count[b]] = nodes
    starts, lens_d = i32([0] + np.cumsum(news).tolist()), i32(lens)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    out, _ = kx.kv_append(kv[0], kv[1], caches[0], caches[1], table, lens_d, starts, i32(count), path=p.cuda() if path else None,
                          max_count=None if path else max(news), k_scale=ks, v_scale=vs, err=err)
    torch.cuda.synchronize()
    assert err.tolist()[0] == 0 and out.tolist() == [a + c for a, c in zip(lens, count)] and lens_d.tolist() == lens
    want = old.double()
    t0 = 0
    for b, n in enumerate(news):
        for i in range(count[b]):
            pos = lens[b] + i
            pg, r = int(table[b, pos // page]), pos % page
            for w, sc in ((0, ks), (1, vs)):
                x = kv[w, :, t0 + int(p[b, i])]
                # the quotient is rounded to FP32 ahead of the code, as the call divides
                want[w, :, pg, r] = x.double() if cache == "bf16" else e4m3((x.float() / sc).double())
        t0 += n
    got = caches.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def test_kv_append_keeps_a_sequence_it_cannot_serve():
    T, page = 9, 16
    kv = torch.randn(2, 2, T, 2, 64, device="cuda").to(BF)
    starts, lens = i32([0, 4, 9]), i32([10, 20])
    base = dict(table=i32([[0, 1], [2, 3]]), count=i32([3, 4]), path=i32([[0, 1, 3, 0], [0, 2, 3, 4]]))

    def go(err_words, **kw):
        caches = torch.zeros(2, 2, 5, page, 2, 64, dtype=BF, device="cuda")
        a = {**base, **kw}
        err = torch.zeros(4, dtype=torch.int32, device="cuda")
        out, _ = kx.kv_append(kv[0], kv[1], caches[0], caches[1], a["table"], a.get("lens", lens), a.get("starts", starts),
                              a["count"], path=a["path"], err=err)
        torch.cuda.synchronize()
        assert err.tolist()[:3] == err_words, (kw, err.tolist())
        return caches, out.tolist()

    good, out = go([0, 0, 0])
    assert out == [13, 24]
    for words, kw, n in (([1, 5, 1], dict(path=i32([[0, 1, 3, 0], [0, 2, 5, 4]])), 20), ([1, -1, 1], dict(path=i32([[0, 1, 3, 0], [-1, 2, 3, 4]])), 20),
                         ([1, 5, 1], dict(table=i32([[0, 1], [2, 5]])), 20), ([1, -3, 1], dict(table=i32([[0, 1], [2, -3]])), 20),
                         ([1, 5, 1], dict(count=i32([3, 5])), 20), ([1, -2, 1], dict(count=i32([3, -2])), 20),
                         ([1, 4, 1], dict(lens=i32([10, 29])), 29)):
        c, out = go(words, **kw)
        assert out == [13, n]
        assert torch.equal(c[:, :, :2], good[:, :, :2]) and (c[:, :, 2:] == 0).all()
    c, out = go([1, 4, 1], starts=i32([0, 4, 12]))
    assert out == [13, 20] and (c[:, :, 2:] == 0).all()


def test_kv_append_after_a_device_acceptance_in_a_graph():
    """The count from mtp_accept's output, chain drafts: nothing comes back to the host in between."""
    kv = torch.randn(2, 6, 1, 128, device="cuda").to(BF)
    caches = torch.zeros(2, 4, 16, 1, 128, dtype=BF, device="cuda")
    cands = torch.zeros(6, 20, 2, dtype=torch.int32, device="cuda")
    cands[:, :, 0] = torch.linspace(9, 1, 20, device="cuda").view(torch.int32)
    cands[:, :, 1] = torch.arange(20, device="cuda") + 100 * torch.arange(6, device="cuda")[:, None]
    nan, drafts = torch.zeros(6, dtype=torch.int32, device="cuda"), i32([0, 100, 200, 7, 400])
    acc = torch.zeros(8, dtype=torch.int32, device="cuda")
    lens, starts, table, lens_out = i32([30]), i32([0, 6]), i32([[2, 0, 3]]), i32([0])

    def step():
        kx.mtp_accept(cands, nan, drafts, None, 0.0, 20, 1.0, 1000, out=acc)
        kx.kv_append(kv[0], kv[1], caches[0], caches[1], table, lens, starts, acc[:1] + 1, max_count=6, lens_out=lens_out)
    step()
    torch.cuda.synchronize()
    assert acc.tolist()[:2] == [3, 0] and lens_out.tolist() == [34]
    ref = caches.clone()
    assert torch.equal(caches[0, 0, 14:16, 0], kv[0, 0:2, 0]) or torch.equal(caches[0, 0, 14:16, 0], kv[0, :2, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        caches.zero_()
        lens_out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(caches, ref) and lens_out.tolist() == [34]


# ---------------- norm ----------------

@pytest.mark.parametrize("act", [BF, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 128), (6, 4096), (7, 640), (33, 2560), (2, 4224), (3, 16384), (2, 32768), (1030, 384), (1100, 2560),
                                 (1025, 4096)])
@pytest.mark.parametrize("residual,w_add", [(False, 0.0), (True, 1.0)])
def test_norm(act, M, K, residual, w_add):
    print(f"norm {act} M={M} K={K} residual={residual}", flush=True)
    g = gen(K + M)
    x = torch.randn(M, K + 8, device="cuda", generator=g).to(act)[:, :K]  # rows apart by more than K
    res = (2 * torch.randn(M, K, device="cuda", generator=g)).to(act) if residual else None
    w = (0.3 * torch.randn(K, device="cuda", generator=g) + (1.0 - w_add)).to(act)
    y = torch.empty(M, K, dtype=act, device="cuda")
    q, scale, rout = kx.add_rms_norm_fp8(x, w, 1e-5, residual=res, w_add=w_add, y=y)
    torch.cuda.synchronize()
    r = x if res is None else (x.float() + res.float()).to(act)
    if res is not None:
        assert torch.equal(rout, r)
    r = r.double()
    wf = (w.float() + w_add).double()  # one FP32 addition
    y64 = r / (r.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * wf
    root = (K / 64 + 16) * U32
    assert ((y.double() - y64).abs() <= ((U16 if act == BF else 16 * U32) + root) * y64.abs()).all()
    runs = y64.view(M, -1, 128)
    peak = runs.abs().amax(2)
    assert ((scale.double() - peak / 448).abs() <= root * peak / 448).all()
    # each code is a nearest one: half a step off, and what FP32 t = r w and its quotient lose (3 u32)
    at = runs * (448 / peak)[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(at.abs().clamp(min=2.0 ** -6))) - 3)
    assert ((q.double().view_as(at) - at).abs() <= step / 2 + 4 * U32 * at.abs()).all()
    if act == BF and w_add == 0.0:  # t is exact: the nearest code of 448 t / amax, ties to even
        t = r * wf
        t = t.view(M, -1, 128)
        want = e4m3((t.abs() * 448 / t.abs().amax(2, keepdim=True)).float().double()) * t.sign()
        assert torch.equal(q.double().view_as(want), want)


def test_norm_odd_values_and_in_place():
    x = torch.randn(4, 512, device="cuda").to(BF)
    w = torch.ones(512, dtype=BF, device="cuda")
    x[1] = 0
    x[2, 130] = float("nan")
    x[3, 256:384] = 0
    q, scale, _ = kx.add_rms_norm_fp8(x, w)
    torch.cuda.synchronize()
    assert (scale[1] == 0).all() and (q[1].float() == 0).all()
    assert torch.isnan(scale[2]).all()
    assert scale[3, 2] == 0 and (q[3, 256:384].float() == 0).all() and (scale[3, [0, 1, 3]] > 0).all()
    tiny = torch.full((1, 128), 2.0 ** -100, dtype=torch.float32, device="cuda")
    tiny[0, 1] = -2.0 ** -101
    q, scale, _ = kx.add_rms_norm_fp8(tiny, torch.ones(128, device="cuda"), eps=0.0)
    assert q[0, 0].float() == 448 and q[0, 1].float() == -224
    a, r = torch.randn(70, 256, device="cuda").to(BF), torch.randn(70, 256, device="cuda").to(BF)
    w = torch.randn(256, device="cuda").to(BF)
    y = torch.empty_like(a)
    want = [t.clone() for t in kx.add_rms_norm_fp8(a, w, residual=r, y=y)]
    a2, r2 = a.clone(), r.clone()
    got = kx.add_rms_norm_fp8(a2, w, residual=r2, residual_out=r2, y=a2)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    assert torch.equal(r2, want[2]) and torch.equal(a2, y)


# ---------------- FP8 linear ----------------

def fp8_case(M, N, K, seed):
    g = gen(seed)
    x = torch.randn(M, K, device="cuda", generator=g).mul_(100).clamp_(-448, 448).to(F8)
    w = torch.randn(N, K, device="cuda", generator=g).mul_(100).clamp_(-448, 448).to(F8)
    xs = torch.rand(M, K // 128, device="cuda", generator=g) * 0.02
    ws = torch.rand(-(-N // 128), K // 128, device="cuda", generator=g) * 0.01
    return x, xs, kx.Fp8Weight(w, ws)


def fp8_reference(x, xs, w):
    xd = x.double() * xs.double().repeat_interleave(128, 1)
    wd = w.q.double() * w.scale.double().repeat_interleave(128, 0)[:w.N].repeat_interleave(128, 1)
    return xd @ wd.T, xd.abs() @ wd.abs().T


@pytest.mark.parametrize("out", [ACT_BF16, ACT_F32])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 128), (1, 4096, 1024), (6, 300, 4096), (16, 129, 640), (5, 77, 1152),       # 16-row blocks
    (17, 1000, 256), (32, 4096, 384), (64, 2000, 2560), (33, 31, 1152),                # 32 x 32 blocks
    (65, 1000, 384), (100, 301, 640), (200, 130, 128), (64, 12288, 256),               # 128 x 64 tiles
    (256, 12288, 256), (250, 12000, 384),                                              # 128 x 128
    (512, 12288, 128), (500, 12301, 256),                                              # 256 x 128
    (1531, 7680, 256), (1530, 7670, 384),                                              # 256 x 192
])
def test_linear_fp8(out, M, N, K):
    print(f"linear_fp8 M={M} N={N} K={K} out={out}", flush=True)
    x, xs, w = fp8_case(M, N, K, seed=M + N)
    guard = torch.full((M * N + 64,), 3.0, dtype=BF if out == ACT_BF16 else torch.float32, device="cuda")
    y = kx.linear_fp8(x, xs, w, out_act=out, y=guard[:M * N].view(M, N))
    torch.cuda.synchronize()
    assert (guard[M * N:] == 3.0).all()
    ref, S = fp8_reference(x, xs, w)
    tol = (K / 32 + 8) * U32 * S if out == ACT_F32 else U16 * ref.abs() + 2.0 ** -12 * S
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.3g} times the tolerance"
    assert float((y.double() - ref).norm() / ref.norm()) <= (1e-6 if out == ACT_F32 else 2.0 ** -8)


def test_linear_fp8_unaligned_output_and_repeat():
    x, xs, w = fp8_case(130, 512, 512, seed=1)
    buf = torch.zeros(130 * 512 + 1, dtype=BF, device="cuda")
    a = kx.linear_fp8(x, xs, w)
    b = kx.linear_fp8(x, xs, w, y=buf[1:].view(130, 512))  # 2-byte aligned
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    c = torch.empty_like(a)
    with torch.cuda.graph(graph):
        kx.linear_fp8(x, xs, w, y=c)
    for _ in range(3):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, c)


def test_linear_fp8_nan_and_zero_scales():
    x, xs, w = fp8_case(20, 200, 512, seed=2)
    xs[3] = 0
    x.view(torch.uint8)[5, 7] = 0x7F
    w.scale[1, 2] = float("nan")
    y = kx.linear_fp8(x, xs, w)
    torch.cuda.synchronize()
    assert torch.isnan(y[5]).all() and torch.isnan(y[:, 128:]).all()
    assert (y[3, :128] == 0).all() and torch.isfinite(y[[0, 1, 2, 4], :128]).all()


# ---------------- scored routing ----------------

def best(x, k):
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    return v[:, :k], i[:, :k]


def route_reference(logits, E, k, score, bias, groups, top, group_best, renorm, factor):
    x = logits[:, :E].double()
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
    c = s if bias is None else s + bias.double()
    if groups > 1:
        v, _ = best(c.view(len(x) * groups, -1), group_best)
        _, chosen = best(v.sum(1).view(len(x), groups), top)
        keep = torch.zeros(len(x), groups, dtype=torch.bool, device="cuda").scatter_(1, chosen, True)
        c = c.masked_fill(~keep.repeat_interleave(E // groups, 1), -math.inf)
    _, ids = best(c, k)
    coef = s.gather(1, ids)
    return ids.to(torch.int32), factor * (coef / coef.sum(1, keepdim=True) if renorm else coef)


@pytest.mark.parametrize("act", [torch.float32, BF])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M,E,k,groups,top,group_best,renorm,biased", [
    (6, 512, 10, 8, 4, 2, True, True), (700, 256, 8, 8, 3, 1, False, True), (5, 160, 6, 8, 3, 1, True, False),
    (3, 1, 1, 1, 1, 1, True, False), (9, 7, 7, 1, 1, 1, False, True), (4, 1024, 32, 1, 1, 1, True, True),
    (8, 64, 8, 8, 1, 2, True, True),       # one group open: every expert of it
    (5, 512, 10, 64, 2, 2, True, False),   # a lane a group, few lanes with open experts
    (6, 1023, 20, 33, 5, 2, False, True),  # 31 experts a lane
    (7, 96, 4, 3, 2, 2, True, True), (2, 512, 32, 2, 1, 1, True, False),
])
def test_scored_routing(act, score, M, E, k, groups, top, group_best, renorm, biased):
    print(f"route M={M} E={E} k={k} {score} groups={groups}", flush=True)
    g = gen(E + k)
    logits = (1.5 * torch.randn(M, E + 3, device="cuda", generator=g)).to(act)  # rows apart by more than E; BF16: ties
    bias = 0.1 * torch.randn(E, device="cuda", generator=g) if biased else None
    if biased and act == BF:
        bias = (bias * 8).round() / 8  # ties past the bias too
    ids, coef, _ = kx.moe_router_scored(logits, E, k, score=score, bias=bias, groups=groups, top_groups=top,
                                        group_best=group_best, renorm=renorm, factor=2.5)
    torch.cuda.synchronize()
    want, ref = route_reference(logits, E, k, score, bias, groups, top, group_best, renorm, 2.5)
    assert torch.equal(ids, want)
    assert ((coef.double() - ref).abs() <= 2 * U32 * ref.abs()).all()


def test_scored_routing_ties_shared_slot_and_errors():
    E, k = 256, 8
    flat = torch.zeros(3, E, device="cuda")  # every score equal: more candidates than a wave ranks at once
    flat[1, 200] = 1.0
    flat[2] = 50.0  # saturated: equal scores of different logits
    flat[2, ::2] = 60.0
    ids, coef, _ = kx.moe_router_scored(flat, E, k, renorm=False)
    assert ids[0].tolist() == list(range(8)) and ids[1].tolist() == [200] + list(range(7)) and ids[2].tolist() == list(range(8))
    ids, _, _ = kx.moe_router_scored(flat[:1], E, k, groups=8, top_groups=2)
    assert ids[0].tolist() == list(range(8))
    logits = torch.randn(4, E + 1, device="cuda")
    shared = logits[:, E]
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    ids, coef, _ = kx.moe_router_scored(logits, E, k, shared=shared, shared_ld=E + 1, shared_id=E, factor=3.0, err=err)
    assert ids.shape == (4, 9) and (ids[:, 8] == E).all() and err.tolist()[0] == 0
    want = torch.sigmoid(shared.double())
    assert ((coef[:, 8].double() - want).abs() <= 4 * U32).all()
    logits[2, 17] = float("inf")
    ids, coef, _ = kx.moe_router_scored(logits, E, k, shared=shared, shared_ld=E + 1, shared_id=E, err=err)
    assert (ids[2] == -1).all() and torch.isnan(coef[2]).all() and (ids[[0, 1, 3]] >= 0).all() and err.tolist()[:3] == [1, 2, 17]
    low = torch.full((1, 16), -800.0, device="cuda")  # scores of zero: the sum too
    ids, coef, _ = kx.moe_router_scored(low, 16, 2)
    assert ids.tolist() == [[0, 1]] and coef.tolist() == [[0.0, 0.0]]


# ---------------- together ----------------

def test_a_verify_layer_with_its_attention():
    """norm and FP8 codes -> FP8 projection -> attention over the cache -> output projection -> norm -> scored routing and
    experts -> head -> acceptance -> append, as a verify runs them; each stage against 64 bits on its own inputs, then the
    whole step again as a captured graph."""
    from strixite_amd import synthetic as syn
    from strixite_amd.verify import MoeVerifyLayer, VerifyAttention, VerifyTail
    d, Hq, Hkv, D, E, I, V = 512, 4, 2, 128, 64, 128, 2000
    b = Batch(D, Hq, Hkv, 16, [37], [6], seed=51)
    b.table = i32([[4, 2, 0, 1]])  # a fourth page for what is appended
    T = 6
    norm_w = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen(1))).to(BF)
    qkv = fp8_case(1, (Hq + 2 * Hkv) * D, d, seed=3)[2]
    qkv.scale.mul_(0.01)
    out_w = syn.qweight(8, d, Hq * D, 64, seed=4)
    att = VerifyAttention(norm_w, qkv, out_w, Hq, Hkv, D, max_tokens=8, max_seqs=2, max_new=8)
    moe = MoeVerifyLayer(syn.router_weight(E, d, seed=5), syn.qweight(4, E * 2 * I, d, 128, seed=6),
                         syn.qweight(4, E * d, I, 128, seed=7), E, 4, 8,
                         routing=dict(score="sigmoid", bias=0.02 * torch.randn(E, device="cuda", generator=gen(8)), groups=8,
                                      top_groups=4, factor=2.0))
    tail = VerifyTail(syn.qweight(8, V, d, 64, seed=9), V, 20, 8)
    x, res = syn.activations(T, d, seed=10), syn.activations(T, d, seed=11)
    mask = kx.tree_mask([list(range(-1, 5))]).cuda()
    drafts = i32([1, 2, 3, 4, 5])
    hid, q2, s2, r2 = (torch.empty(T, d, dtype=BF, device="cuda"), torch.empty(T, d, dtype=F8, device="cuda"),
                       torch.empty(T, d // 128, device="cuda"), torch.empty(T, d, dtype=BF, device="cuda"))
    lens_out = i32([0])

    def step():
        y, r = att.forward(x, res, b.kc, b.vc, b.table, b.lens, b.starts, mask)
        kx.add_rms_norm_fp8(y, norm_w, 1e-6, residual=r, residual_out=r2, y=hid, q=q2, scale=s2)
        h = moe.forward(hid)
        acc = tail.forward(h, drafts, None, 0.0, 20, 1.0)
        kx.kv_append(att.k_new, att.v_new, b.kc, b.vc, b.table, b.lens, b.starts, acc[:1] + 1, max_count=6, lens_out=lens_out)
        return y, h, acc

    kc, vc = b.kc.clone(), b.vc.clone()
    y, h, acc = step()
    torch.cuda.synchronize()
    # the projection from its own codes
    ref, S = fp8_reference(att.q8[:T], att.scale[:T], qkv)
    assert ((att.heads[:T].reshape(T, -1).double() - ref).abs() <= U16 * ref.abs() + 2.0 ** -12 * S).all()
    # the attention from its own heads
    b.q, b.kn, b.vn = att.heads[:T].split([Hq, Hkv, Hkv], dim=1)
    b.mask, b.max_new, after_k, after_v = mask, 8, b.kc, b.vc
    b.kc, b.vc = kc, vc
    check(b, att.att[:T])
    assert torch.equal(r2, (y.float() + att.residual[:T].float()).to(BF))
    ids, coef = route_reference(moe.logits[:T], E, 4, "sigmoid", moe.routing["bias"], 8, 4, 2, True, 2.0)
    assert torch.equal(moe.ids[:T], ids) and ((moe.coef[:T].double() - coef).abs() <= 2 * U32 * coef).all()
    assert torch.isfinite(h.float()).all() and moe.expert_err.tolist()[0] == 0 and att.err.tolist()[0] == 0
    j = int(acc[0])
    assert lens_out.tolist() == [38 + j] and int(acc[1]) == 0
    for i in range(j + 1):
        p = 37 + i
        assert torch.equal(after_k[int(b.table[0, p // 16]), p % 16], att.k_new[i])
        assert torch.equal(after_v[int(b.table[0, p // 16]), p % 16], att.v_new[i])
    # captured: the same bits, replay after replay
    b.kc, b.vc = kc.clone(), vc.clone()
    want = [t.clone() for t in (y, h, acc)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # the stream's own workspace and sync buffers
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        b.kc.copy_(kc), b.vc.copy_(vc)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))
        assert torch.equal(b.kc, after_k) and torch.equal(b.vc, after_v)


def test_two_graphs_with_one_workspace_replayed_in_turn():
    """Nothing in a workspace outlives a call: graphs of different shapes that share one, on one stream, with eager work
    between the replays, give what each gives alone."""
    a, b = Batch(128, 8, 2, 32, [700, 3], [5, 1], seed=61), Batch(128, 8, 2, 16, [90], [24], seed=62)
    want = [x.run()[0].clone() for x in (a, b)]
    n = max(kx.tree_attention_workspace_bytes(x.lens.numel(), 8, 2, 128, x.max_new) for x in (a, b))
    ws = torch.empty((n + 7) // 8, dtype=torch.int64, device="cuda")
    outs, graphs = [], []
    for x in (a, b):
        outs.append(torch.empty_like(x.q))
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1]):
            x.run(ws=ws, out=outs[-1])
    for turn in range(4):
        for i in ((0, 1) if turn % 2 else (1, 0)):
            outs[i].zero_()
            ws.fill_(-1)
            graphs[i].replay()
            assert torch.equal(outs[i], want[i]), (turn, i)


def test_verify_attention_with_a_rotation_on_another_stream():
    from strixite_amd import synthetic as syn
    from strixite_amd.verify import VerifyAttention
    d, Hq, Hkv, D = 512, 4, 2, 128
    b = Batch(D, Hq, Hkv, 16, [37], [6], seed=63)
    mask = kx.tree_mask([list(range(-1, 5))]).cuda()
    qkv = fp8_case(1, (Hq + 2 * Hkv) * D, d, seed=64)[2]
    qkv.scale.mul_(0.01)
    streams = []

    def rotate(q, k):
        streams.append(torch.cuda.current_stream().cuda_stream)
        q.neg_(), k.mul_(0.5)  # exact
    att = VerifyAttention(torch.ones(d, dtype=BF, device="cuda"), qkv, syn.qweight(8, d, Hq * D, 64, seed=65), Hq, Hkv, D, 8, 2, 8,
                          rotate=rotate)
    x = syn.activations(6, d, seed=66)
    want = att.forward(x, None, b.kc, b.vc, b.table, b.lens, b.starts, mask)[0].clone()
    heads = att.heads[:6].clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = att.forward(x, None, b.kc, b.vc, b.table, b.lens, b.starts, mask, stream=s)[0]
    s.synchronize()
    assert streams[1] == s.cuda_stream != streams[0]
    assert torch.equal(att.heads[:6], heads) and torch.equal(got, want)


# ---------------- attention: FP16 P, many sequences ----------------

@pytest.mark.parametrize("D,G,news", [(64, 2, 1), (128, 4, 6), (128, 8, 8), (128, 8, 12), (128, 8, 24), (64, 8, 32), (256, 8, 3),
                                      (256, 8, 8), (256, 8, 16), (256, 8, 32)])
def test_attention_fp8_keeps_a_long_tail_under_a_peak(D, G, news):
    """The first key 2^26 over the 2047 others of its sequence, which hold all of the values: in units of the peak each is
    under FP16's smallest number, together they are the output. FP16 P loses 2^-25 a key on a sum of 2^7: keys 2^-32 max |v|;
    the rest as above. Enough sequences and heads that a block takes whole ones."""
    print(f"attention fp8 tail D={D} G={G} news={news}", flush=True)
    page, L, B, Hkv = 128, 2048, 64, 8
    pages = L // page
    kc, vc = (torch.zeros(pages, page, Hkv, D, device="cuda") for _ in range(2))
    vc[:] = 0.5 + torch.rand(Hkv, D, device="cuda", generator=gen(D))
    kc[0, 0, :, 0], vc[0, 0] = 18.0, 0.0
    T = B * news
    q = torch.zeros(T, Hkv * G, D, dtype=BF, device="cuda")
    q[:, :, 0] = 1.0
    new = torch.ones(T, Hkv, D, dtype=BF, device="cuda")
    lse = torch.empty(T, Hkv * G, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(B, 1)
    out, _ = kx.tree_attention(q, new, new, kc.to(F8), vc.to(F8), table, i32([L] * B), i32(list(range(0, T + 1, news))),
                               torch.zeros(T, 1, dtype=torch.int64, device="cuda"), news, scale=1.0, lse=lse)
    v = vc[0, 1].to(F8).double().repeat_interleave(G, 0)
    tail = (L - 1) * math.exp(-18.0)
    want = v * tail / (1 + tail)
    e = (D + 4) * U32 * 18.0
    tol = U16 * want + (2.0 ** -11 + 2 * e + (L + 64) * U32) * want + L * 2.0 ** -32 * v.max()
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())
    assert ((lse.double() - (18.0 + math.log1p(tail))).abs() <= e + (L + 64) * U32 + 4 * U32 * 18.0).all()


@pytest.mark.parametrize("D,Hq,news", [(128, 4, [6]), (128, 8, [12]), (64, 8, [24]), (256, 8, [6]), (256, 8, [20])])
def test_attention_fp8_rising_maxima(D, Hq, news):
    """Scores that rise by tens through a long FP8 cache: FP16 P never leaves its range."""
    print(f"attention fp8 rising D={D} Hq={Hq} news={news}", flush=True)
    b = Batch(D, Hq, 1, 64, [9001], news, "fp8", seed=6, amp=3.0)
    k = b.kc.view(-1, 1, D)
    b.kc = (k.float() * torch.linspace(0.1, 2.0, k.shape[0], device="cuda").view(-1, 1, 1)).to(F8).view_as(b.kc)
    b.table = torch.arange(b.table.numel(), dtype=torch.int32, device="cuda").view_as(b.table)
    check(b, b.run()[0])


def many(D, Hq, Hkv, B, most, cache, seed):
    """B sequences of up to 90 cached and `most` drafted tokens, some of them with none of either."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 91, (B,), generator=g)
    news = torch.randint(0, 4, (B,), generator=g)
    lens[torch.rand(B, generator=g) < 0.1] = 0
    lens[B // 2], news[B // 2], news[B // 3], news[-1] = 90, most, most, 1
    return Batch(D, Hq, Hkv, 16, lens.tolist(), news.tolist(), cache, seed=seed, mask="any")


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
@pytest.mark.parametrize("D,Hq,Hkv,B,most", [
    (64, 24, 8, 40, 3), (64, 40, 8, 40, 20), (128, 12, 4, 40, 5), (128, 40, 8, 33, 20), (256, 10, 2, 70, 6), (256, 24, 8, 40, 40),
    (64, 3, 1, 64, 2),                                                                    # a row a lane group, heads left over
    (128, 4, 2, 600, 3), (64, 6, 3, 1024, 9), (128, 8, 2, 1000, 64), (256, 2, 1, 257, 4),  # several sequences a thread
])
def test_attention_many_short_sequences(D, Hq, Hkv, B, most, cache):
    """More sequences than an eighth of the blocks: the join gives every row a lane group of its own."""
    print(f"attention many D={D} {cache} Hq={Hq} Hkv={Hkv} B={B} most={most}", flush=True)
    b = many(D, Hq, Hkv, B, most, cache, seed=B + D)
    lse = torch.empty(b.T, Hq, device="cuda")
    out, err = b.run(lse=lse, err=torch.zeros(4, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert err.tolist()[0] == 0
    check(b, out, lse)


@pytest.mark.parametrize("D,Hq,Hkv,B", [(64, 24, 8, 40), (128, 12, 4, 40), (256, 10, 2, 70), (128, 4, 2, 600)])
def test_attention_one_unreadable_sequence_among_many(D, Hq, Hkv, B):
    print(f"attention unreadable D={D} B={B}", flush=True)
    b = many(D, Hq, Hkv, B, 7, "bf16", seed=B)
    o, tol, l, ltol = b.reference()
    i = B // 2
    rows = torch.zeros(b.T, dtype=torch.bool, device="cuda")
    rows[int(b.starts[i]):int(b.starts[i + 1])] = True
    room = b.table.shape[1] * 16
    for word, at in ((room + 1, "lens"), (-5, "lens"), (b.kc.shape[0], "page")):
        where = b.lens[i:i + 1] if at == "lens" else b.table[i, 1:2]
        keep = where.clone()
        where.fill_(word)
        lse, err = torch.zeros(b.T, Hq, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
        out = b.run(lse=lse, err=err)[0].double()
        torch.cuda.synchronize()
        assert err.tolist()[:3] == [1, word, i]
        assert torch.isnan(out[rows]).all() and torch.isnan(lse[rows]).all()
        assert ((out - o).abs() <= tol)[~rows].all()
        none = l.isinf()
        assert torch.equal(lse.isinf()[~rows], none[~rows])
        ok = ~rows[:, None] & ~none
        assert ((lse.double() - l).abs() <= ltol)[ok].all()
        where.copy_(keep)
    check(b, b.run()[0])


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
@pytest.mark.parametrize("layers,Hkv,D,page,lens,news", [
    (2, 2, 64, 16, [5, 0, 130], [700, 1, 257]),
    (1, 1, 128, 64, [63], [2049]),
    (3, 8, 128, 256, [0, 255], [513, 300]),
])
def test_kv_append_of_prompt_chunks(cache, layers, Hkv, D, page, lens, news):
    """Whole chunks without a path, hundreds of tokens over many pages; what lies beside them stays."""
    print(f"append chunk {cache} layers={layers} D={D} lens={lens} news={news}", flush=True)
    host = torch.Generator().manual_seed(D)
    B, T = len(lens), sum(news)
    P = max(-(-(a + n) // page) for a, n in zip(lens, news))
    table = torch.randperm(B * P + 2, generator=host)[:B * P].to(torch.int32).view(B, P).cuda()
    kv = (2 * torch.randn(2, layers, T, Hkv, D, device="cuda", generator=gen(D))).to(BF)
    old = torch.randn(2, layers, B * P + 2, page, Hkv, D, device="cuda", generator=gen(D + 1)).to(BF if cache == "bf16" else F8)
    ks, vs = (1.0, 1.0) if cache == "bf16" else (0.0625, 0.125)  # powers of two: the quotients are exact
    got, starts, err = old.clone(), i32([0] + np.cumsum(news).tolist()), torch.zeros(4, dtype=torch.int32, device="cuda")
    out, _ = kx.kv_append(kv[0], kv[1], got[0], got[1], table, i32(lens), starts, i32(news), max_count=max(news), k_scale=ks,
                          v_scale=vs, err=err)
    torch.cuda.synchronize()
    assert err.tolist()[0] == 0 and out.tolist() == [a + n for a, n in zip(lens, news)]
    want = old.double().view(2, layers, -1, Hkv, D)
    t0 = 0
    for b, (a, n) in enumerate(zip(lens, news)):
        pos = torch.arange(a, a + n, device="cuda")
        slot = table[b].long()[pos // page] * page + pos % page
        x = kv[:, :, t0:t0 + n].double()
        if cache == "fp8":
            x = e4m3(torch.stack([x[0] / ks, x[1] / vs]))
        want[:, :, slot] = x
        t0 += n
    assert torch.equal(got.double().view_as(want), want)


def test_verify_attention_on_two_streams_at_once():
    from strixite_amd import synthetic as syn
    from strixite_amd.verify import VerifyAttention
    d, Hq, Hkv, D = 512, 4, 2, 128
    b = Batch(D, Hq, Hkv, 16, [900], [6], seed=71)
    mask = kx.tree_mask([list(range(-1, 5))]).cuda()
    qkv = fp8_case(1, (Hq + 2 * Hkv) * D, d, seed=72)[2]
    qkv.scale.mul_(0.01)
    att = VerifyAttention(torch.ones(d, dtype=BF, device="cuda"), qkv, syn.qweight(8, d, Hq * D, 64, seed=73), Hq, Hkv, D, 8, 2, 8)
    xs = [syn.activations(6, d, seed=74 + i) for i in range(2)]
    go = lambda x, s=None: att.forward(x, x, b.kc, b.vc, b.table, b.lens, b.starts, mask, stream=s)
    want = [[t.clone() for t in (*go(x), att.k_new)] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [(*go(x, s), att.k_new) for x, s in zip(xs, streams)]
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(w, g))


@pytest.mark.parametrize("M", [6, 40, 100, 600])  # rows, rows of 32, the tiles
def test_linear_fp8_where_large_products_cancel(M):
    """+-448 * 448 beside small products inside a block. BF16 outputs: a product loses less than 2^-13 of the largest power of
    two 2^(ex + ew) among its eight neighbours (codes under 2^-6 as 2^-6), so 8 of that a group, and the output's rounding; FP32
    outputs (K / 32 + 8) u32 S, as ever. The group's own sums: (K / 8 + 8) u32 S."""
    print(f"linear_fp8 cancelling M={M}", flush=True)
    N, K = 256, 256
    g = gen(M)
    code = lambda r: (torch.randn(r, K, device="cuda", generator=g) * 100 *
                      2.0 ** torch.randint(-12, 1, (r, K), device="cuda", generator=g)).clamp(-448, 448).to(F8).float()
    x, w = code(M), code(N)
    x[:, 8::32], x[:, 9::32] = 448, 448
    w[:, 8::32], w[:, 9::32] = 448, -448
    x[0, :], x[0, 8:10] = 7.5, 448            # one group: six of 7.5, each just under the cut beside the pair
    w[0, :], w[0, 8], w[0, 9], w[0, 10:16] = 0, 448, -448, 1
    one = torch.ones(N // 128, K // 128, device="cuda")
    weight, xs = kx.Fp8Weight(w.to(F8), one), torch.ones(M, K // 128, device="cuda")
    ref, S = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
    power = lambda t: torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6)))
    cut = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for k in range(0, K, 8):
        cut += 2.0 ** -10 * torch.exp2((power(x[:, None, k:k + 8]) + power(w[None, :, k:k + 8])).amax(2)).double()
    y = kx.linear_fp8(x.to(F8), xs, weight).double()
    assert ((y - ref).abs() <= U16 * ref.abs() + cut + (K / 8 + 8) * U32 * S).all()
    y = kx.linear_fp8(x.to(F8), xs, weight, out_act=ACT_F32).double()
    assert ((y - ref).abs() <= (K / 32 + 8) * U32 * S).all() and float(y[0, 0]) == 45.0
