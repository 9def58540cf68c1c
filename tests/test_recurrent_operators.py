"""The gated delta rule, the acceptance by probabilities, the 8-bit integer linear and the norms around a block without a GPU: host
checks of the C entries, and the packed structures against the C layouts."""
import ctypes
import struct

import pytest
import torch

import strixite_amd as sx
from strixite_amd import kernels as kx


@pytest.fixture(scope="module")
def L():
    return sx.lib()


BUF = (ctypes.c_uint8 * (1 << 20))()
BASE = (ctypes.addressof(BUF) + 255) // 256 * 256


def P(off=0):
    return None if off is None else ctypes.c_void_p(BASE + off)


def refused(L, rc, text):
    msg = L.sx_last_error().decode()
    assert rc == sx.SX_EINVAL and text in msg, (rc, msg)


def test_packed_structures_have_the_c_layout():
    vals = list(range(1, 12)) + [0] + list(range(13, 32)) + [0.5]
    d = sx.DeltaC.from_buffer_copy(kx._DELTA(*vals))
    flat = []
    for name, _ in d._fields_:
        x = getattr(d, name)
        flat += [x.p, x.token, x.head, x.layer or 0] if isinstance(x, sx.HeadRows) else [x]
    assert [f or 0 for f in flat] == vals
    vals = list(range(1, 15)) + [0.5, 0.25, 0.125, 2.0]
    n = sx.BlockNormC.from_buffer_copy(kx._NORM(*vals))
    assert [getattr(n, f[0]) for f in n._fields_] == vals
    assert ctypes.sizeof(sx.DeltaC) == struct.calcsize("@PqqqPqqqPqqqPPqqPPPPPqqqqqqqqiif4x")


# q, k [4, 2, 64] and v [4, 4, 64] slices of one buffer; two states
def delta(**kw):
    rows = lambda o: sx.HeadRows(BASE + o, 512, 64, 0)
    d = dict(q=rows(0), k=rows(256), v=rows(512), a=BASE + 8192, b=BASE + 8448, a_token=4, b_token=4, A_log=BASE + 8704, dt_bias=BASE + 8768,
             state=BASE + 65536, slot=BASE + 8832, starts=BASE + 8896, T=4, key_heads=2, heads=4, key_dim=64, dim=64, slots=2, state_slot=16384,
             batch=2, gate_act=sx.ACT_BF16, normalize=1, scale=0.125)
    d.update(kw)
    return sx.DeltaC(**d)


def run(L, max_len=4, out=(16384, 256, 64), ws=None, ws_bytes=0, **kw):
    o = sx.HeadRows(BASE + out[0], out[1], out[2], 0)
    return L.sx_gated_delta(ctypes.byref(delta(**kw)), max_len, ctypes.byref(o), P(ws), ws_bytes, None, None)


def verify(L, max_new=4, mask_ld=1, out=(16384, 256, 64), u=20480, decay=32768, mask=33024, **kw):
    o = sx.HeadRows(BASE + out[0], out[1], out[2], 0)
    return L.sx_gated_delta_verify(ctypes.byref(delta(**kw)), max_new, P(mask), mask_ld, ctypes.byref(o), P(u), P(decay), None, None)


BAD_DELTA = [
    (dict(a=None), "null pointer"), (dict(state=None), "null pointer"), (dict(A_log=None), "go together"), (dict(gate_act=7), "gate dtype"),
    (dict(T=0), "T = 0"), (dict(batch=0), "batch"), (dict(batch=1025), "batch"), (dict(key_heads=3), "multiple of the key heads"),
    (dict(heads=1), "multiple of the key heads"), (dict(heads=2048, key_heads=2), "up to 1024"), (dict(key_dim=96), "key_dim"), (dict(dim=40), "dim = 40"),
    (dict(dim=0), "dim = 0"), (dict(slots=0), "slots"), (dict(slot=None, slots=1), "slots = 1"), (dict(state_slot=16380), "state_slot"),
    (dict(state_slot=16386), "state_slot"), (dict(state=BASE + 65540), "16-byte"), (dict(q=sx.HeadRows(BASE + 2, 512, 64, 0)), "16-byte"),
    (dict(k=sx.HeadRows(BASE, 508, 64, 0)), "multiples of 8"), (dict(v=sx.HeadRows(BASE, -512, 64, 0)), "multiples of 8"), (dict(a=BASE + 8193), "aligned"),
    (dict(b_token=-1), "gate strides"), (dict(q=sx.HeadRows(BASE, 1 << 25, 64, 0)), "up to 2^24"), (dict(out=(16384, 1 << 25, 64)), "up to 2^24"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(out=(16384, 250, 64)), "multiples of 4"), (dict(out=(16388, 256, 64)), "8-byte aligned"), (dict(out=(16384, 256, 32)), "heads that overlap"),
    (dict(out=(512, 512, 64)), "overlaps q, k or v"), (dict(out=(8192, 256, 64)), "overlaps the gates"), (dict(out=(65536, 256, 64)), "overlaps the states"),
]


@pytest.mark.parametrize("kw,text", BAD_DELTA + [
    (dict(max_len=0), "max_len"), (dict(max_len=17), "workspace of 0"), (dict(max_len=17, ws=196608 + 4, ws_bytes=1 << 30), "16-byte aligned"),
    (dict(max_len=17, ws=65536, ws_bytes=1 << 30), "workspace overlaps"), (dict(state=BASE + 512), "overlaps"), (dict(state=BASE, out=(262144, 256, 64)), "state overlaps q"),
])
def test_gated_delta_refusals(L, kw, text):
    refused(L, run(L, **kw), text)


@pytest.mark.parametrize("kw,text", BAD_DELTA + [
    (dict(max_new=0), "max_new"), (dict(max_new=65), "max_new"), (dict(mask_ld=0), "mask_ld"), (dict(mask=33028), "misaligned"), (dict(u=20484), "16-byte"),
    (dict(u=512), "u overlaps q, k or v"), (dict(decay=8896), "decay overlaps starts"), (dict(u=65536), "overlap"), (dict(decay=20480), "overlap"),
    (dict(u=16384), "overlap"), (dict(mask=20480), "overlap"),
])
def test_gated_delta_verify_refusals(L, kw, text):
    refused(L, verify(L, **kw), text)


def commit(L, k=(0, 512, 64, 0), u=16384, decay=24576, layers=1, T=4, Hk=2, Hv=4, Dk=64, Dv=64, state=65536, state_layer=0, state_slot=16384, slots=2,
           slot=8832, starts=8896, batch=2, count=8960, max_count=4, path=9024, path_ld=4):
    rows = sx.HeadRows(BASE + k[0], *k[1:])
    return L.sx_gated_delta_commit(ctypes.byref(rows), P(u), P(decay), layers, T, Hk, Hv, Dk, Dv, P(state), state_layer, state_slot, slots, P(slot), P(starts),
                                   batch, P(count), max_count, P(path), path_ld, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(u=None), "null pointer"), (dict(count=None), "null pointer"), (dict(layers=0), "layers"), (dict(batch=0), "batch"), (dict(Hv=3), "multiple of the key heads"),
    (dict(Dk=32), "key_dim"), (dict(Dv=24), "dim = 24"), (dict(max_count=65, path_ld=65), "max_count"), (dict(max_count=0), "max_count"), (dict(path_ld=3), "path_ld"),
    (dict(slot=None, slots=1), "slots"), (dict(k=(0, 516, 64, 0)), "multiples of 8"), (dict(state_slot=100), "state strides"), (dict(layers=2), "states overlap"),
    (dict(layers=2, state_layer=16384), "states overlap"), (dict(state=65544), "16-byte"), (dict(u=65536), "overlap another"), (dict(count=65536), "overlap another"),
    (dict(slot=65600), "overlap another"),
])
def test_gated_delta_commit_refusals(L, kw, text):
    refused(L, commit(L, **kw), text)


def test_gated_delta_workspace(L):
    n = ctypes.c_size_t()
    size = lambda *a: (L.sx_gated_delta_workspace_bytes(*a, ctypes.byref(n)), n.value)
    assert size(16, 4, 2, 4, 128, 16) == (0, 0)
    rc, a = size(640, 4, 2, 4, 128, 17)
    assert rc == 0 and a > 0 and a % 16 == 0
    assert size(1280, 4, 2, 4, 128, 17)[1] > a and size(640, 4, 2, 4, 64, 17)[1] < a
    for bad in ((0, 4, 2, 4, 128, 17), (640, 0, 2, 4, 128, 17), (640, 4, 3, 4, 128, 17), (640, 4, 2, 4, 96, 17), (640, 4, 2, 4, 128, 0)):
        refused(L, size(*bad)[0], "key_dim")
    assert kx.gated_delta_workspace_bytes(640, 4, 2, 4, 128, 17) == a


def linear(L, x=0, xs=4096, q=8192, ws=16384, N=40, K=112, y=32768, M=4, act=sx.ACT_BF16):
    v = sx.Int8View(None if q is None else BASE + q, BASE + ws, N, K)
    return L.sx_linear_int8(P(x), P(xs), ctypes.byref(v), P(y), M, act, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null pointer"), (dict(q=None), "null pointer"), (dict(K=100), "multiple of 16"), (dict(K=0), "multiple of 16"), (dict(K=131072), "131056"),
    (dict(N=0), "weight [0"), (dict(M=0), "M = 0"), (dict(M=1 << 23), "M = "), (dict(act=2), "output dtype"), (dict(x=8), "16-byte"), (dict(q=8200), "16-byte"),
    (dict(y=32769), "to its elements"), (dict(y=64), "y overlaps"), (dict(y=16384), "y overlaps"), (dict(N=0x7ffffff0, M=1 << 22), "too many tiles"),
])
def test_linear_int8_refusals(L, kw, text):
    refused(L, linear(L, **kw), text)


def norm(L, M=4, K=256, act=sx.ACT_BF16, **kw):
    off = dict(x=0, post=8192, gate=16384, residual=24576, pre=32768, residual_out=40960, y=49152, q=57344, scale=65536)
    d = dict(ldx=256, ld_gate=256, group=0, post_len=0, gate_act=0, eps=1e-6, w_add=0.0, residual_scale=1.0, branch_scale=1.0)
    for k, v in kw.items():
        (off if k in off else d)[k] = v
    s = sx.BlockNormC(**{k: None if v is None else BASE + v for k, v in off.items()}, **d)
    return L.sx_block_norm_int8(ctypes.byref(s), M, K, act, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null pointer"), (dict(q=None, y=None, scale=None, residual=None, residual_out=None), "no output"), (dict(q=None), "go together"),
    (dict(residual=None), "go together"), (dict(act=5), "activation dtype"), (dict(M=0), "M = 0"), (dict(K=20), "multiple of 8"), (dict(K=16392), "16384"),
    (dict(ldx=248), "ldx"), (dict(ldx=260), "ldx"), (dict(ld_gate=8), "ld_gate"), (dict(ld_gate=300), "ld_gate"), (dict(gate_act=3), "gate activation"),
    (dict(group=96), "group = 96"), (dict(group=4), "group = 4"), (dict(group=1024), "group"), (dict(post_len=128), "post_len"), (dict(eps=float("nan")), "eps"),
    (dict(branch_scale=float("inf")), "branch_scale"), (dict(x=8), "16-byte"), (dict(q=57348), "8-byte"), (dict(y=256), "other rows"), (dict(y=8192), "other rows"),
    (dict(x=0, ldx=512, y=0), "other rows"), (dict(scale=57344), "overlap"), (dict(residual_out=49152), "overlap"), (dict(q=24576), "other rows"),
    (dict(ld_gate=0, y=16384), "other rows"),
])
def test_block_norm_refusals(L, kw, text):
    refused(L, norm(L, **kw), text)


def accept(L, logits=0, ld=100, T=6, V=100, draft=4096, dld=100, Vd=80, act=sx.ACT_F32, drafts=8192, starts=8256, B=2, rows=4, u=8320, temp=8448,
           tokens=8512, count=8576, status=8640, ws=16384, ws_bytes=1 << 16):
    return L.sx_mtp_accept_sampled(P(logits), ld, T, V, P(draft), dld, Vd, act, P(drafts), P(starts), B, rows, P(u), P(temp), P(tokens), P(count), P(status),
                                   P(ws), ws_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(logits=None), "null pointer"), (dict(u=None), "null pointer"), (dict(act=2), "logit dtype"), (dict(T=0), "T = 0"), (dict(T=40000), "T = "),
    (dict(B=0), "batch"), (dict(B=1025), "batch"), (dict(V=0), "n_valid"), (dict(ld=99), "ld = 99"), (dict(draft=None), "go together"), (dict(Vd=0), "go together"),
    (dict(Vd=101, dld=101), "n_draft"), (dict(dld=79), "draft_ld"), (dict(rows=0), "max_rows"), (dict(rows=257), "max_rows"), (dict(ws_bytes=100), "workspace of 100"),
    (dict(ws=16388), "16-byte aligned"), (dict(u=8324), "to their elements"), (dict(tokens=0), "overlaps an input"), (dict(count=8512), "overlap"),
    (dict(status=8256), "overlaps an input"), (dict(ws=0), "overlaps an input"),
])
def test_accept_refusals(L, kw, text):
    refused(L, accept(L, **kw), text)


def test_accept_workspace(L):
    n = ctypes.c_size_t()
    assert L.sx_mtp_accept_sampled_workspace_bytes(6, 2, 5000, 0, ctypes.byref(n)) == 0
    without = n.value
    assert L.sx_mtp_accept_sampled_workspace_bytes(6, 2, 5000, 5000, ctypes.byref(n)) == 0 and n.value > 2 * without > 0
    refused(L, L.sx_mtp_accept_sampled_workspace_bytes(6, 2, 50, 51, ctypes.byref(n)), "n_draft = 51")


def test_python_calls_refuse_tensors_on_the_host():
    t = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    q, k, v, a = t(3, 1, 64), t(3, 1, 64), t(3, 1, 64), t(3, 1)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    state = torch.zeros(1, 1, 64, 64)
    for f in (lambda: kx.gated_delta(q, k, v, a, a, state, i(2), 3), lambda: kx.gated_delta_verify(q, k, v, a, a, state, i(2), torch.zeros(3, 1, dtype=torch.int64), 3),
              lambda: kx.gated_delta_commit(k, torch.zeros(3, 1, 64), torch.zeros(3, 1), state, i(2), i(1), max_count=3),
              lambda: kx.block_norm_int8(t(2, 64)), lambda: kx.mtp_accept_sampled(t(2, 9), i(2), i(2), torch.zeros(2, 2, dtype=torch.float64), torch.zeros(1), 2),
              lambda: kx.linear_int8(torch.zeros(1, 16, dtype=torch.int8), torch.zeros(1), kx.Int8Weight(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)))):
        with pytest.raises(sx.SxError, match="not on a GPU"):
            f()
