"""The attention half of a verify layer and scored routing without a GPU: host checks of the C entries and of the Python
functions, the mask builder, and the packed structures against the C layouts."""
import ctypes
import struct

import pytest
import torch

import strixite_amd as sx
from strixite_amd import kernels as kx


@pytest.fixture(scope="module")
def L():
    return sx.lib()


BUF = (ctypes.c_uint8 * (1 << 16))()
BASE = (ctypes.addressof(BUF) + 255) // 256 * 256


def P(off=0):
    return ctypes.c_void_p(BASE + off)


def refused(L, rc, text):
    msg = L.sx_last_error().decode()
    assert rc == sx.SX_EINVAL and text in msg, (rc, msg)


def test_packed_structures_have_the_c_layout():
    vals = (1, 2, 1, 0.5, 0.25, *range(5, 18), 77, 78, 79, 80, 81)
    c = sx.KvCacheC.from_buffer_copy(kx._CACHE(*vals))
    assert [getattr(c, f[0]) for f in c._fields_] == list(vals)
    r = sx.HeadRows.from_buffer_copy(kx._ROWS(9, 8, 7, 6))
    assert (r.p, r.token, r.head, r.layer) == (9, 8, 7, 6)
    assert ctypes.sizeof(sx.KvCacheC) == struct.calcsize("@2Pi2f5q8qP2qPq")


def test_tree_mask():
    m = kx.tree_mask([[-1, 0, 0, 1], [-1], [-1, -1, 1]])
    assert m.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b1], [0b1], [0b10], [0b110]]
    chain = kx.tree_mask([list(range(-1, 69))])
    assert chain.shape == (70, 2) and chain[63].tolist() == [-1, 0] and chain[69].tolist() == [-1, 0b111111]
    with pytest.raises(ValueError):
        kx.tree_mask([[0]])
    with pytest.raises(ValueError):
        kx.tree_mask([[-1, -2]])


def cache(**kw):
    d = dict(k=BASE, v=BASE + 4096, dtype=sx.KV_BF16, k_scale=1.0, v_scale=1.0, pages=4, page_size=16, heads=2, dim=64,
             layers=1, k_page=2048, k_token=128, k_head=64, k_layer=0, v_page=2048, v_token=128, v_head=64, v_layer=0,
             table=BASE + 8192, table_ld=2, pages_per_seq=2, lens=BASE + 8448, batch=2)
    d.update(kw)
    return sx.KvCacheC(**d)


def attention(L, c=None, T=4, Hq=4, max_new=4, mask_ld=1, scale=0.1, q=(0, 256, 64), out=(16384, 256, 64), ws=1 << 40, ptr=None):
    c = c or cache()
    rows = lambda o, t, h: ctypes.byref(sx.HeadRows(BASE + o, t, h, 0))
    return L.sx_tree_attention(rows(*q), rows(2048, 128, 64), rows(4096, 128, 64), T, Hq, ctypes.byref(c), P(9000 // 8 * 8),
                               max_new, P(9216), mask_ld, scale, rows(*out), None, ptr or P(12288), ws, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(c=dict(page_size=24)), "power of two"), (dict(c=dict(page_size=8)), "power of two"),
    (dict(c=dict(dim=96)), "head dimension"), (dict(Hq=5), "multiple of the key heads"), (dict(Hq=1), "multiple"),
    (dict(max_new=257, mask_ld=5), "max_new"), (dict(max_new=0), "max_new"), (dict(max_new=65), "mask_ld"),
    (dict(T=0), "T = 0"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(c=dict(batch=1025)), "1..1024"), (dict(c=dict(batch=0)), "batch"), (dict(c=dict(pages=0)), "pages"),
    (dict(c=dict(k_token=130)), "multiples of 16 bytes"), (dict(c=dict(k=BASE + 8)), "16-byte aligned"),
    (dict(c=dict(dtype=2)), "cache dtype"), (dict(c=dict(dtype=1, v_scale=0.0)), "v_scale"),
    (dict(c=dict(table_ld=1)), "table_ld"), (dict(c=dict(k=None)), "null pointer"), (dict(c=dict(layers=2)), "one layer"),
    (dict(c=dict(k_token=1 << 27)), "2^31"), (dict(q=(2, 256, 64)), "16-byte aligned"),
    (dict(q=(0, 252, 64)), "multiples of 8"), (dict(q=(0, 256, 32)), "heads overlap"), (dict(out=(128, 256, 64)), "out overlaps"),
    (dict(ws=1000), "workspace of 1000"), (dict(ptr=P(12296)), "16-byte aligned"),
])
def test_tree_attention_refusals(L, kw, text):
    kw = dict(kw)
    if isinstance(kw.get("c"), dict):
        kw["c"] = cache(**kw["c"])
    refused(L, attention(L, **kw), text)


def append(L, c=None, T=4, max_count=2, path=None, path_ld=0, lens_out=9984, layer=0):
    c = c or cache()
    rows = lambda o: ctypes.byref(sx.HeadRows(BASE + o, 128, 64, layer))
    return L.sx_kv_append(rows(0), rows(2048), T, ctypes.byref(c), P(9000 // 8 * 8), P(9216), max_count, path, path_ld,
                          P(lens_out), None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(T=0), "T = 0"), (dict(max_count=0), "max_count"), (dict(max_count=70000), "max_count"),
    (dict(path=P(9600), path_ld=1), "path_ld"), (dict(lens_out=8448), "lens_out overlaps"), (dict(layer=12), "layer strides"),
    (dict(c=dict(dim=60)), "dim = 60"), (dict(c=dict(page_size=17)), "power of two"),
])
def test_kv_append_refusals(L, kw, text):
    kw = dict(kw)
    if isinstance(kw.get("c"), dict):
        kw["c"] = cache(**kw["c"])
    refused(L, append(L, **kw), text)


def norm(L, x=0, ldx=256, residual=None, weight=8192, M=4, K=256, eps=1e-6, w_add=0.0, residual_out=None, y=None, q=16384,
         scale=20480, act=sx.ACT_BF16):
    p = lambda o: None if o is None else P(o)
    return L.sx_add_rms_norm_fp8(p(x), ldx, p(residual), p(weight), M, K, eps, w_add, p(residual_out), p(y), p(q), p(scale),
                                 act, None)


@pytest.mark.parametrize("kw,text", [
    (dict(K=200), "multiple of 128"), (dict(K=32896, ldx=32896), "32768"), (dict(ldx=248), "ldx"), (dict(ldx=260), "ldx"),
    (dict(M=0), "M = 0"), (dict(q=None, scale=None), "no output"), (dict(scale=None), "go together"),
    (dict(residual=4096), "go together"), (dict(eps=-1.0), "eps"), (dict(w_add=float("inf")), "w_add"), (dict(act=7), "dtype 7"),
    (dict(x=2), "aligned"), (dict(y=512), "overlaps an input"), (dict(q=256), "overlaps"), (dict(y=8192), "weight"),
    (dict(residual=4096, residual_out=12288, y=12288), "y overlaps residual_out"),
])
def test_norm_refusals(L, kw, text):
    refused(L, norm(L, **kw), text)


def fp8(L, x=0, xs=4096, q=8192, ws=16384, y=20480, M=4, N=16, K=256, out=sx.ACT_BF16):
    w = sx.Fp8View(BASE + q if q is not None else None, BASE + ws, N, K)
    return L.sx_linear_fp8(P(x), P(xs), ctypes.byref(w), P(y), M, out, None)


@pytest.mark.parametrize("kw,text", [
    (dict(K=192), "multiple of 128"), (dict(K=1 << 17), "65536"), (dict(M=0), "M = 0"), (dict(N=0), "weight [0"),
    (dict(out=5), "output dtype 5"), (dict(x=8), "aligned"), (dict(y=20481), "aligned"), (dict(y=0), "overlaps"),
    (dict(y=16384), "overlaps"), (dict(q=None), "null pointer"), (dict(M=(1 << 22) + 1), "M ="),
])
def test_linear_fp8_refusals(L, kw, text):
    refused(L, fp8(L, **kw), text)


def route(L, ld=64, M=2, E=64, k=4, score=sx.SCORE_SIGMOID, groups=8, top=4, best=2, factor=1.0, shared=None, sld=1, sid=0,
          act=sx.ACT_F32, ids=8192, coef=12288):
    return L.sx_moe_router_scored(P(), ld, M, E, k, score, None, groups, top, best, 1, factor, shared, sld, sid, P(ids),
                                  P(coef), act, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(E=1025, ld=1025), "E = 1025"), (dict(k=33), "k = 33"), (dict(k=0), "k = 0"), (dict(ld=63), "ld = 63"),
    (dict(score=2), "unknown score"), (dict(groups=7), "divisor"), (dict(groups=128), "groups"), (dict(top=9), "top_groups"),
    (dict(k=9, top=1), "chosen groups"), (dict(groups=64, best=2), "group_best"), (dict(best=3), "group_best"),
    (dict(factor=float("inf")), "factor"), (dict(shared=P(), sid=-1), "shared_id"), (dict(shared=P(), sld=0), "shared_ld"),
    (dict(act=3), "dtype 3"), (dict(M=0), "M = 0"), (dict(coef=8192), "same buffer"),
])
def test_scored_routing_refusals(L, kw, text):
    refused(L, route(L, **kw), text)


def test_workspace_bytes(L):
    n = ctypes.c_size_t()
    assert L.sx_tree_attention_workspace_bytes(3, 8, 2, 128, 6, ctypes.byref(n)) == 0 and n.value > 0
    refused(L, L.sx_tree_attention_workspace_bytes(3, 8, 3, 128, 6, ctypes.byref(n)), "multiple of the key heads")
    refused(L, L.sx_tree_attention_workspace_bytes(3, 8, 2, 100, 6, ctypes.byref(n)), "head dimension")


def test_python_refuses_what_is_not_on_a_gpu_or_does_not_fit():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16)
    with pytest.raises(sx.SxError, match="not on a GPU"):
        kx.add_rms_norm_fp8(x, w)
    with pytest.raises(sx.SxError, match="multiple of 128"):
        kx.add_rms_norm_fp8(x[:, :200], w[:200])
    with pytest.raises(TypeError):
        kx.add_rms_norm_fp8(x.half(), w)
    with pytest.raises(sx.SxError, match="multiple of 128"):
        kx.Fp8Weight(torch.zeros(16, 100, dtype=torch.float8_e4m3fn), torch.ones(1, 1))
    with pytest.raises(sx.SxError, match="scale must be"):
        kx.Fp8Weight(torch.zeros(200, 256, dtype=torch.float8_e4m3fn), torch.ones(1, 2))
    weight = kx.Fp8Weight(torch.zeros(200, 256, dtype=torch.float8_e4m3fn), torch.ones(2, 2))
    with pytest.raises(sx.SxError, match="not on a GPU"):
        kx.linear_fp8(torch.zeros(2, 256, dtype=torch.float8_e4m3fn), torch.ones(2, 2), weight)
    with pytest.raises(sx.SxError, match="not one of"):
        kx.moe_router_scored(torch.zeros(2, 64), 64, 4, score="tanh")
    with pytest.raises(sx.SxError, match="for E ="):
        kx.moe_router_scored(torch.zeros(2, 64), 65, 4)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    kv = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    table = i32(0, 1, 2, 3).view(2, 2)
    mask = torch.ones(3, 1, dtype=torch.int64)
    with pytest.raises(sx.SxError, match="not on a GPU"):
        kx.tree_attention(q, kv, kv, c, c, table, i32(1, 2), i32(0, 1, 3), mask, 2)
    with pytest.raises(sx.SxError, match="not on a GPU"):
        kx.kv_append(kv, kv, c, c, table, i32(1, 2), i32(0, 1, 3), i32(1, 1), max_count=1)


def test_verify_attention_rotates_on_the_stream_of_its_kernels(monkeypatch):
    from contextlib import contextmanager

    from strixite_amd import verify
    current, seen = ["its caller's"], []

    @contextmanager
    def on(stream):
        before, current[0] = current[0], stream or current[0]
        yield
        current[0] = before

    for f in ("add_rms_norm_fp8", "linear_fp8", "tree_attention", "linear"):
        monkeypatch.setattr(verify.kx, f, lambda *a, stream=None, **kw: seen.append(stream or current[0]))
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(verify.VerifyAttention, "_ws_for", lambda self, stream: None)

    class W:
        N, K = 128, 128

    class Qkv:
        N, K = 384, 128
    att = verify.VerifyAttention(torch.ones(128), Qkv, W, 2, 2, 64, 4, 1, 4, rotate=lambda q, k: seen.append(current[0]))
    x, lens = torch.zeros(4, 128), torch.zeros(1, dtype=torch.int32)
    att.forward(x, None, None, None, None, lens, None, None, stream="its own")
    assert seen == ["its own"] * 5
    seen.clear()
    att.forward(x, None, None, None, None, lens, None, None)
    assert seen == ["its caller's"] * 5


def test_workspace_and_err_have_to_hold_what_is_written(monkeypatch):
    """Before anything reaches the library: what the strides or the size of a buffer would let a kernel write beside it."""
    def unreached(*a, **kw):
        raise AssertionError("the call went on")
    monkeypatch.setattr(kx, "_together", lambda dev, tensors: None)
    monkeypatch.setattr(kx, "_run", unreached)
    q, kv = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    table, mask, ws = i32(0, 1, 2, 3).view(2, 2), torch.ones(3, 1, dtype=torch.int64), torch.zeros(64, dtype=torch.int64)
    att = lambda **kw: kx.tree_attention(q, kv, kv, c, c, table, i32(1, 2), i32(0, 1, 3), mask, 2, **{"ws": ws, **kw})
    with pytest.raises(sx.SxError, match="ws must be contiguous"):
        att(ws=ws[::2])
    for err in (i32(0), torch.zeros(4), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(sx.SxError, match="err must be"):
            att(err=err)
        with pytest.raises(sx.SxError, match="err must be"):
            kx.kv_append(kv, kv, c, c, table, i32(1, 2), i32(0, 1, 3), i32(1, 1), max_count=1, err=err)
        with pytest.raises(sx.SxError, match="err must be"):
            kx.moe_router_scored(torch.zeros(2, 64), 64, 4, err=err)


def test_a_workspace_made_for_a_call_belongs_to_the_stream_of_the_call(monkeypatch):
    from contextlib import contextmanager
    current, made = ["its caller's"], []

    @contextmanager
    def on(stream):
        before, current[0] = current[0], stream or current[0]
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(kx, "_together", lambda dev, tensors: None)
    monkeypatch.setattr(kx, "_run", lambda *a, **kw: None)
    monkeypatch.setattr(kx, "tree_attention_workspace", lambda *a: made.append(current[0]) or torch.zeros(8, dtype=torch.int64))
    q, kv = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    for stream in ("its own", None):
        kx.tree_attention(q, kv, kv, c, c, i32(0, 1, 2, 3).view(2, 2), i32(1, 2), i32(0, 1, 3),
                          torch.ones(3, 1, dtype=torch.int64), 2, stream=stream)
    assert made == ["its own", "its caller's"]


@pytest.mark.parametrize("lens_out", [8192, 8196, 9000 // 8 * 8, 9004, 9216, 9220, 9600, 9612])
def test_append_refuses_lens_out_in_what_its_blocks_read(L, lens_out):
    refused(L, append(L, path=P(9600), path_ld=2, lens_out=lens_out), "lens_out overlaps")


@pytest.mark.parametrize("strides", [(0, 64), (192, 64), (64, 128), (64, 192)])
def test_attention_refuses_an_output_whose_rows_share_memory(L, strides):
    refused(L, attention(L, ws=100, out=(16384, *strides)), "rows of out share memory")


@pytest.mark.parametrize("strides", [(256, 64), (64, 256), (512, 128), (128, 512), (128, 64 + 448)])
def test_attention_takes_an_output_whose_rows_are_apart(L, strides):
    refused(L, attention(L, ws=100, out=(16384, *strides)), "workspace of 100")  # the next check


def test_attention_refuses_a_workspace_in_its_output(L):
    n = ctypes.c_size_t()
    assert L.sx_tree_attention_workspace_bytes(2, 4, 2, 64, 4, ctypes.byref(n)) == sx.SX_OK
    refused(L, attention(L, ws=n.value, ptr=P(16384 + 256)), "workspace overlap")


@pytest.mark.parametrize("kw", [dict(k_page=0), dict(v_page=2040), dict(k_token=64), dict(v_token=0), dict(layers=2),
                                dict(layers=2, k_layer=8192, v_layer=2048)])
def test_append_refuses_a_cache_whose_rows_share_memory(L, kw):
    refused(L, append(L, c=cache(**kw)), "rows of the cache share memory")


@pytest.mark.parametrize("kw", [dict(layers=2, k_layer=8192, v_layer=8192), dict(k_page=2048, k_token=64, k_head=1024),
                                dict(layers=2, k_layer=2048, k_page=4096, v_layer=2048, v_page=4096), dict(pages=1, k_page=0)])
def test_append_takes_layers_heads_and_pages_in_any_order(L, kw):
    refused(L, append(L, c=cache(**kw), max_count=0), "max_count = 0")  # the next check


@pytest.mark.parametrize("kw,text", [(dict(coef=8192 + 28), "same buffer or overlap"), (dict(ids=508), "overlap the logits"),
                                     (dict(coef=0), "overlap the logits")])
def test_routing_refuses_outputs_in_its_logits_or_each_other(L, kw, text):
    refused(L, route(L, **kw), text)


def test_routing_refuses_a_shared_stride_past_the_tensor(monkeypatch):
    calls = []
    monkeypatch.setattr(kx, "_together", lambda dev, tensors: None)
    monkeypatch.setattr(kx, "_run", lambda *a, **kw: calls.append(a))
    logits = torch.zeros(3, 65)
    go = lambda shared, ld: kx.moe_router_scored(logits, 64, 4, shared=shared, shared_ld=ld, shared_id=64)
    with pytest.raises(sx.SxError, match="leads past"):
        go(torch.zeros(3), 65)
    with pytest.raises(sx.SxError, match="leads past"):
        go(logits[:, 64], 66)
    go(torch.zeros(3), 1), go(logits[:, 64], 65)
    assert len(calls) == 2


class Streams:
    """Stands in for torch's streams and devices on the CPU: `now` is the stream that torch would call current, `made` the
    one that was current at each torch.empty."""

    class Stream:
        def __init__(self, n):
            self.cuda_stream = n

    def __init__(self, monkeypatch):
        from contextlib import contextmanager, nullcontext
        self.default, self.now, self.made = self.Stream(0), self.Stream(0), []
        empty = torch.empty

        @contextmanager
        def on(stream):
            before, self.now = self.now, stream or self.now
            yield
            self.now = before
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch.cuda, "device", lambda d: nullcontext())
        monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: self.now)
        monkeypatch.setattr(torch, "empty", lambda *a, **kw: self.made.append(self.now.cuda_stream) or empty(*a, **kw))
        like, new = torch.empty_like, torch.Tensor.new_empty
        monkeypatch.setattr(torch, "empty_like", lambda *a, **kw: self.made.append(self.now.cuda_stream) or like(*a, **kw))
        monkeypatch.setattr(torch.Tensor, "new_empty", lambda *a, **kw: self.made.append(self.now.cuda_stream) or new(*a, **kw))
        for f in ("zeros", "full"):  # made and filled
            monkeypatch.setattr(torch, f, lambda *a, real=getattr(torch, f), **kw: self.made.append(self.now.cuda_stream) or real(*a, **kw))
        fill = torch.Tensor.fill_
        monkeypatch.setattr(torch.Tensor, "fill_", lambda *a: self.made.append(self.now.cuda_stream) or fill(*a))


class Weight:
    """The shape of an attention layer's weights, without them: 2 + 2 + 2 heads of 64 over 128 features."""

    def __init__(self, N):
        self.N, self.K = N, 128


def attention_layer():
    from strixite_amd import verify
    return verify.VerifyAttention(torch.ones(128), Weight(384), Weight(128), 2, 2, 64, 4, 1, 4)


def test_a_workspace_that_a_layer_keeps_belongs_to_its_stream(monkeypatch):
    streams, layer = Streams(monkeypatch), attention_layer()
    streams.made.clear()
    layer._ws_for(Streams.Stream(7))
    assert streams.made and set(streams.made) == {7}
    streams.made.clear()
    layer._ws_for(Streams.Stream(7))
    assert streams.made == []
    with torch.cuda.stream(Streams.Stream(9)):
        layer._ws_for(None)
    assert streams.made and set(streams.made) == {9}


def test_forwards_of_a_layer_on_two_streams_share_no_buffer(monkeypatch):
    from strixite_amd import verify
    streams, written = Streams(monkeypatch), []
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
    outs = dict(add_rms_norm_fp8=("residual_out", "q", "scale"), linear_fp8=("y",), tree_attention=("out", "ws"), linear=("y",))
    for f, names in outs.items():
        monkeypatch.setattr(verify.kx, f, lambda *a, names=names, **kw: written.extend(span(kw[n]) for n in names))
    layer, x, lens = attention_layer(), torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    layer_parts = ("residual", "q8", "scale", "heads", "att", "y")

    def forward(stream):
        written.clear()
        y, r = layer.forward(x, x, None, None, None, lens, None, None, stream=stream)
        assert y.data_ptr() == layer.y.data_ptr() and r.data_ptr() == layer.residual.data_ptr()
        assert layer.k_new.data_ptr() == layer.heads[:, 2].data_ptr()
        return list(written), [span(getattr(layer, n)) for n in layer_parts]
    one, two = Streams.Stream(1), Streams.Stream(2)
    (a, parts_a), (b, parts_b), (again, _) = forward(one), forward(two), forward(one)
    assert len(a) == 7 and a == again
    assert all(lo2 >= hi1 or lo1 >= hi2 for lo1, hi1 in a + parts_a for lo2, hi2 in b + parts_b)
    with torch.cuda.stream(two):
        assert forward(None)[0] == b


def operator_calls():
    """Each of the five operators on small tensors, without the buffers that it can make, and how many it makes then."""
    bf, f8 = torch.bfloat16, torch.float8_e4m3fn
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    x, q = torch.zeros(3, 128, dtype=bf), torch.zeros(3, 4, 64, dtype=bf)
    kv, c = torch.zeros(3, 2, 64, dtype=bf), torch.zeros(4, 16, 2, 64, dtype=bf)
    w = kx.Fp8Weight(torch.zeros(16, 128, dtype=torch.uint8).view(f8), torch.ones(1, 1))
    codes, scale = torch.zeros(3, 128, dtype=torch.uint8).view(f8), torch.ones(3, 1)
    seqs = (i32(0, 1, 2, 3).view(2, 2), i32(1, 2), i32(0, 1, 3))
    mask, logits = torch.ones(3, 1, dtype=torch.int64), torch.zeros(3, 64)
    return {
        "norm": (3, lambda s: kx.add_rms_norm_fp8(x, x[0], residual=x, stream=s)),
        "linear": (1, lambda s: kx.linear_fp8(codes, scale, w, stream=s)),
        "attention": (2, lambda s: kx.tree_attention(q, kv, kv, c, c, *seqs, mask, 2, stream=s)),
        "append": (1, lambda s: kx.kv_append(kv, kv, c, c, *seqs, i32(1, 1), max_count=1, stream=s)),
        "routing": (2, lambda s: kx.moe_router_scored(logits, 64, 4, stream=s)),
    }


@pytest.mark.parametrize("name", ["norm", "linear", "attention", "append", "routing"])
def test_buffers_that_a_call_makes_belong_to_its_stream(monkeypatch, name):
    n, call = operator_calls()[name]
    streams = Streams(monkeypatch)
    monkeypatch.setattr(kx, "_together", lambda dev, tensors: None)
    monkeypatch.setattr(kx, "_run", lambda *a, **kw: None)
    monkeypatch.setattr(kx, "tree_attention_workspace_bytes", lambda *a: 64)
    call(Streams.Stream(3))
    assert streams.made == [3] * n
    streams.made.clear()
    call(None)
    assert streams.made == [0] * n


def earlier_calls():
    """The other operators that make buffers: the arguments are placeholders, nothing is launched."""
    x, ids = torch.zeros(2, 64), torch.zeros(2, 3, dtype=torch.int32)
    w, e = Weight(64), Weight(8 * 64)
    w.bits, w.G, w.q, w.scale, w.minv, w.view = 8, 64, torch.zeros(64 * 128, dtype=torch.uint8), ids, ids, lambda: None
    e.view = w.view
    big = torch.zeros(2, 3, 2, dtype=torch.int32)
    return {
        "linear": lambda s: kx.linear(x, w, stream=s),
        "experts_gather": lambda s: kx.experts_gather(x, e, 8, ids, stream=s),
        "experts_combine": lambda s: kx.experts_combine(x, e, 8, ids, x, stream=s),
        "moe_router": lambda s: kx.moe_router(x, 8, 3, stream=s),
        "router_group": lambda s: kx.router_group(x, 8, 3, stream=s),
        "verify_gate_up": lambda s: kx.verify_gate_up(x, x, e, 8, 3, stream=s),
        "verify_down": lambda s: kx.verify_down(x, e, ids, x, 8, stream=s),
        "verify_layer": lambda s: kx.verify_layer(x, x, e, e, 8, 3, ids, stream=s),
        "group_routes": lambda s: kx.group_routes(ids, 8, stream=s),
        "gather_grouped": lambda s: kx.gather_grouped(x, e, 8, ids, 2, 3, stream=s),
        "combine_grouped": lambda s: kx.combine_grouped(x, e, 8, ids, x, ids, stream=s),
        "swiglu": lambda s: kx.swiglu(x, stream=s),
        "linear_f32w": lambda s: kx.linear_f32w(x, x, stream=s),
        "linear_bf16w": lambda s: kx.linear_bf16w(x, x, stream=s),
        "logits_topk": lambda s: kx.logits_topk(x, 64, stream=s),
        "logits_topk_noalloc": lambda s: kx.logits_topk_noalloc(x, 64, stream=s),
        "quantize_q4_from_q8": lambda s: kx.quantize_q4_from_q8(w, stream=s),
        "mtp_pick": lambda s: kx.mtp_pick(x, ids, ids, ids, ids, stream=s),
        "verify_tail": lambda s: kx.verify_tail(x, 64, 3, ids, drafts=ids[0], stream=s),
        "mtp_accept": lambda s: kx.mtp_accept(big, ids, ids[0, :1], None, 0.0, 3, 1.0, 64, stream=s),
    }


@pytest.mark.parametrize("name", list(earlier_calls()))
def test_buffers_of_the_other_operators_belong_to_the_call_s_stream(monkeypatch, name):
    class Library:
        def __getattr__(self, name):
            return lambda *a: 0
    call = earlier_calls()[name]
    streams = Streams(monkeypatch)
    monkeypatch.setattr(kx, "lib", Library)
    call(Streams.Stream(3))
    assert streams.made and set(streams.made) == {3}
    made = len(streams.made)
    call(None)
    assert streams.made[made:] == [0] * made


def test_a_sync_buffer_that_a_layer_keeps_is_zeroed_on_its_stream(monkeypatch):
    from strixite_amd import verify
    streams = Streams(monkeypatch)
    layer = verify.MoeVerifyLayer.__new__(verify.MoeVerifyLayer)
    layer._syncs, layer._dev = {}, torch.device("cpu")
    layer._sync_for(Streams.Stream(4))
    assert streams.made == [4]


FAR = 1 << 24  # behind all that the caches of these tests span; nothing is read there


def append_far(L, **kw):
    """kv_append with everything but the caches out of their way."""
    a = dict(k=FAR, v=FAR + 4096, strides=(128, 64, 0), starts=FAR + 8192, count=FAR + 8448, lens_out=FAR + 8704, err=None)
    a.update({n[4:]: v for n, v in kw.items() if n.startswith("new_")})
    c = cache(**{"table": BASE + FAR + 9216, "lens": BASE + FAR + 9472, **{n: v for n, v in kw.items() if not n.startswith("new_")}})
    rows = lambda o: ctypes.byref(sx.HeadRows(BASE + o, *a["strides"]))
    p = lambda o: None if o is None else P(o)
    return L.sx_kv_append(rows(a["k"]), rows(a["v"]), 4, ctypes.byref(c), p(a["starts"]), p(a["count"]), 2, None, 0,
                          p(a["lens_out"]), p(a["err"]), None)
@pytest.mark.parametrize("kw", [
    dict(v=BASE), dict(v=BASE + 128),                                                # the keys' own, a row on
    dict(v=BASE + 4096 - 256),                                                       # into the second page
    dict(k=BASE + 128, v=BASE, k_token=192, v_token=192, k_page=4096, v_page=4096),  # interleaved rows that reach into each other
    dict(v=BASE + 256, k_token=256, k_page=4096, v_page=4096),                       # beside each other, steps that differ
    dict(layers=2, k_layer=16384, v_layer=8192),                                     # the second layer's values over the pages
])
def test_append_refuses_caches_of_keys_and_values_that_share_memory(L, kw):
    refused(L, append_far(L, **{**dict(v=BASE + 4 * 4096), **kw}), "keys and values share memory")


@pytest.mark.parametrize("kw", [
    dict(v=BASE + 4 * 4096), dict(k=BASE + 4 * 4096, v=BASE),                        # one behind the other
    dict(v=BASE + 4096, k_page=4096, v_page=4096),                                   # [pages, 2, page, heads, dim]
    dict(k=BASE + 4096, v=BASE, k_page=4096, v_page=4096, v_token=64, v_head=1024),  # the same, heads outermost in the values
    dict(v=BASE + 256, k_page=4096, v_page=4096, k_token=256, v_token=256),          # [pages, page, 2, heads, dim]
    dict(v=BASE + 128, k_page=4096, v_page=4096, k_token=256, v_token=256, k_head=128, v_head=128),  # [.., heads, 2, dim]
    dict(layers=3, v=BASE + 16384, k_layer=16384, v_layer=16384),                    # [layers, 2, pages, ..]
    dict(layers=3, v=BASE + 4096, k_page=12288, v_page=12288, k_layer=4096, v_layer=4096),  # [pages, layers, 2, ..]
    dict(v=BASE + 16, dtype=sx.KV_E4M3, dim=16, k_head=32, v_head=32, k_token=64, v_token=64),
])
def test_append_takes_keys_and_values_in_one_buffer(L, kw):
    refused(L, append_far(L, new_err=FAR + 9, **kw), "4-byte aligned")  # the last check


@pytest.mark.parametrize("kw", [
    dict(new_k=0), dict(new_v=128), dict(new_k=16384 + 4096), dict(new_v=16384 + 8192), dict(new_k=2 * 16384 - 128),
    dict(new_k=16384 - 1024, new_strides=(128, 64, 0)),                                    # its last row is a row of the values
    dict(layers=2, k_layer=32768, v_layer=32768, new_k=8192, new_strides=(128, 64, 16384)),  # in the pages of every layer
])
def test_append_refuses_new_rows_in_the_cache(L, kw):
    refused(L, append_far(L, v=BASE + 16384, **kw), "lies in the cache")


@pytest.mark.parametrize("kw", [
    dict(new_k=2 * 16384, new_v=2 * 16384 + 1024),
    dict(layers=2, k_layer=32768, v_layer=32768, new_k=32768, new_v=33792, new_strides=(128, 64, 32768)),  # a slab a layer: pages, rows
])
def test_append_takes_new_rows_beside_the_cache(L, kw):
    refused(L, append_far(L, v=BASE + 16384, new_err=FAR + 9, **kw), "4-byte aligned")  # the last check


def attention_far(L, T=4, err=FAR + 9, **at):
    """tree_attention with everything apart: offsets of its arguments, those of out with strides."""
    a = dict(q=(0, 256, 64), k_new=(4096, 128, 64), v_new=(8192, 128, 64), k=16384, v=32768, table=49152, lens=49664, starts=50176,
             mask=50688, out=(53248, 256, 64), lse=57344, ws=FAR)
    a.update(at)
    c = cache(k=BASE + a["k"], v=BASE + a["v"], table=BASE + a["table"], lens=BASE + a["lens"])
    rows = lambda n: ctypes.byref(sx.HeadRows(BASE + a[n][0], *a[n][1:], 0))
    return L.sx_tree_attention(rows("q"), rows("k_new"), rows("v_new"), T, 4, ctypes.byref(c), P(a["starts"]), 4, P(a["mask"]), 1,
                               0.1, rows("out"), P(a["lse"]), P(a["ws"]), 1 << 40, P(err), None)


def test_attention_takes_arguments_that_lie_apart(L):
    refused(L, attention_far(L), "4-byte aligned")  # the last check
    # one buffer of [tokens, query | key | value | output heads, 64]
    refused(L, attention_far(L, q=(0, 768, 64), k_new=(512, 768, 64), v_new=(768, 768, 64), out=(1024, 768, 64)), "4-byte aligned")


@pytest.mark.parametrize("kw", [
    *[dict(out=(o, 256, 64)) for o in (16384, 32768 + 8192, 49152, 49664, 50176 - 1920, 50688, 50704)],
    *[dict(lse=o) for o in (0, 2044, 4096, 8192 + 1020, 16384, 49148, 49152, 49668, 50180, 50684, 50712)],
    *[dict(ws=o) for o in (0, 4096, 8192, 49152, 49664, 50176, 50688, -4096)],
    dict(T=3, q=(0, 512, 64), out=(768, 512, 64)),               # in one buffer, its last head the next token's q
])
def test_attention_refuses_outputs_in_what_it_reads(L, kw):
    rc, msg = attention_far(L, **kw), L.sx_last_error().decode()
    assert rc == sx.SX_EINVAL and "overlap" in msg, msg


@pytest.mark.parametrize("kw", [dict(starts=50178), dict(lens=49666), dict(table=49153), dict(lse=57346), dict(err=FAR + 2)])
def test_attention_refuses_misaligned_words(L, kw):
    refused(L, attention_far(L, **{"err": FAR + 8, **kw}), "4-byte aligned")


def route_far(L, logits=32768, ids=8192, coef=12288, bias=16384, shared=20480, sld=1, M=64, k=4, err=FAR + 1, act=sx.ACT_F32):
    return L.sx_moe_router_scored(P(logits), 64, M, 64, k, sx.SCORE_SIGMOID, P(bias), 1, 1, 1, 1, 1.0, P(shared), sld, 64, P(ids),
                                  P(coef), act, P(err), None)


@pytest.mark.parametrize("kw,text", [
    (dict(bias=12288 + 64 * 5 * 4 - 4), "overlap the bias"), (dict(bias=8192 - 252), "overlap the bias"), (dict(ids=16384), "overlap the bias"),
    (dict(shared=8192), "overlap the shared"), (dict(shared=12288 - 63 * 4 * 8, sld=8, ids=FAR), "overlap the shared"),
    (dict(coef=20480 + 252), "overlap the shared"),
    (dict(), "4-byte aligned"),  # apart: the last check
    *[({n: o, "err": FAR}, "4-byte aligned") for n, o in
      (("ids", 8194), ("coef", 12289), ("bias", 16386), ("shared", 20482), ("logits", 32770))],
])
def test_routing_refuses_outputs_in_its_bias_or_shared_logits(L, kw, text):
    refused(L, route_far(L, **kw), text)


def test_verify_attention_runs_on_its_device_whichever_is_current(monkeypatch):
    from contextlib import contextmanager

    from strixite_amd import verify
    current, seen = [0], []

    @contextmanager
    def on(device):
        before, current[0] = current[0], torch.device(device).index
        yield
        current[0] = before

    class OnGpu1:  # in the place of the norm's weight
        is_cuda = True
    streams, layer = Streams(monkeypatch), attention_layer()
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(verify.VerifyAttention, "_ws_for", lambda self, stream: None)
    for f in ("add_rms_norm_fp8", "linear_fp8", "tree_attention", "linear"):
        monkeypatch.setattr(verify.kx, f, lambda *a, **kw: seen.append(current[0]))
    layer.norm_w, layer._dev, layer.rotate = OnGpu1, torch.device("cuda", 1), lambda q, k: seen.append(current[0])
    args = (torch.zeros(4, 128), None, None, None, None, torch.zeros(1, dtype=torch.int32), None, None)
    layer.forward(*args)
    layer.forward(*args, stream=streams.default)
    assert seen == [1] * 10 and current == [0]


@pytest.mark.parametrize("M,routing", [(3, dict(score="softmax")), (3, None), (2000, None)])
def test_moe_verify_layer_runs_on_its_device_whichever_is_current(monkeypatch, M, routing):
    from contextlib import contextmanager

    from strixite_amd import verify
    current, seen = [0], []

    @contextmanager
    def on(device):
        before, current[0] = current[0], torch.device(device).index
        yield
        current[0] = before

    class OnGpu1:  # in the place of the router's weight
        is_cuda = True
    gate_up, down = Weight(4 * 256), Weight(4 * 128)
    layer = verify.MoeVerifyLayer(torch.zeros(4, 128), gate_up, down, 4, 2, M, routing=routing)
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    for f in ("linear_f32w", "moe_router_scored", "group_routes", "router_group", "moe_router", "gather_grouped", "combine_grouped"):
        monkeypatch.setattr(verify.kx, f, lambda *a, **kw: seen.append(current[0]))
    monkeypatch.setattr(verify.MoeVerifyLayer, "_fused", lambda self, M: False)
    layer.Wr, layer._dev = OnGpu1, torch.device("cuda", 1)
    layer.forward(torch.zeros(M, 128))
    assert len(seen) >= 4 and set(seen) == {1} and current == [0]


@pytest.mark.parametrize("bad", [1e-45, 2.9e-39, 2.0 ** -101, 2.0 ** 101, float("inf"), float("nan"), -1.0])
def test_scales_of_a_cache_that_fp32_cannot_divide_by_are_refused(L, bad):
    for kw in (dict(k_scale=bad), dict(v_scale=bad)):
        refused(L, attention(L, c=cache(dtype=sx.KV_E4M3, **kw), ws=100), "expected 2^-100..2^100")
        refused(L, append(L, c=cache(dtype=sx.KV_E4M3, **kw), max_count=0), "expected 2^-100..2^100")
        refused(L, attention(L, c=cache(**kw), ws=100), "workspace of 100")  # a BF16 cache has none
    edge = dict(k_scale=2.0 ** -100, v_scale=2.0 ** 100)
    refused(L, attention(L, c=cache(dtype=sx.KV_E4M3, **edge), ws=100), "workspace of 100")


@pytest.mark.parametrize("scale,k_scale,dtype", [(1e-45, 1.0, sx.KV_BF16), (3e38, 1.0, sx.KV_BF16), (1e-10, 2.0 ** -99, sx.KV_E4M3),
                                                 (1e10, 2.0 ** 100, sx.KV_E4M3)])
def test_a_scale_of_scores_outside_the_normal_numbers_is_refused(L, scale, k_scale, dtype):
    refused(L, attention(L, c=cache(dtype=dtype, k_scale=k_scale), scale=scale, ws=100), "a normal number")


@pytest.mark.parametrize("D,Hq,Hkv,max_new,dtype,keys", [  # keys: a stage's, by the tile that the rows take
    (256, 8, 1, 8, sx.KV_BF16, 32), (256, 8, 1, 8, sx.KV_E4M3, 64), (256, 4, 1, 8, sx.KV_BF16, 64), (128, 4, 1, 8, sx.KV_BF16, 128),
    (128, 8, 1, 8, sx.KV_BF16, 64), (128, 8, 1, 8, sx.KV_E4M3, 128), (64, 4, 1, 8, sx.KV_E4M3, 256), (64, 4, 1, 256, sx.KV_BF16, 256),
])
def test_attention_counts_the_stages_of_its_tile(L, D, Hq, Hkv, max_new, dtype, keys):
    groups = -(-max_new * Hq // 256)
    for pages, ok in ((2 ** 30 // 1024 // 16 * keys // groups, True), (2 ** 31 // 1024 // 16 * keys // groups, False)):
        e, far = (1 if dtype else 2), 1 << 44
        if pages * 16 > 2 ** 31 - 65536 - 16:
            continue  # no sequence is that long
        c = cache(dtype=dtype, k=BASE + far, v=BASE + 2 * far, heads=Hkv, dim=D, k_page=16 * D, v_page=16 * D, k_token=D, v_token=D,
                  k_head=D, v_head=D, table=BASE + 3 * far, table_ld=pages, pages_per_seq=pages, lens=BASE + 4 * far, batch=1024)
        rows = lambda o, t: ctypes.byref(sx.HeadRows(BASE + o, t, D, 0))
        rc = L.sx_tree_attention(rows(0, Hq * D), rows(1 << 24, D), rows(2 << 24, D), 4, Hq, ctypes.byref(c), P(3 << 24), max_new,
                                 P(4 << 24), 4, 0.1, rows(5 << 24, Hq * D), None, P(6 << 24), 1 << 40, P(1), None)
        refused(L, rc, "4-byte aligned" if ok else "more than 2^31 units")


def test_attention_refuses_more_rows_than_its_second_launch_has_blocks(L):
    refused(L, attention(L, T=1 << 24, ws=100), "expected 1..16777215")
    refused(L, attention(L, T=(1 << 24) - 1, ws=100, out=(1 << 40, 256, 64)), "workspace of 100")


@pytest.mark.parametrize("kw", [dict(new_starts=FAR + 8193), dict(new_count=FAR + 8450), dict(new_lens_out=FAR + 8707), dict(table=BASE + FAR + 9218),
                                dict(lens=BASE + FAR + 9473), dict(new_err=FAR + 9)])
def test_append_refuses_misaligned_words(L, kw):
    refused(L, append_far(L, v=BASE + 16384, **{"new_err": FAR + 9728, **kw}), "4-byte aligned")
