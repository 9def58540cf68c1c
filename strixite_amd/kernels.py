"""Python face of the C ABI over torch device tensors: the reference's strix::kernels operators by name
(kernels/linear_q4.hpp, linear_q8.hpp, moe_router.hpp, moe_grouped.hpp, swiglu.hpp, logits_topk.hpp, mtp_pick.hpp).

torch supplies device memory and the stream (torch.cuda.current_stream() unless one is passed); every computation is
a libstrixite_amd.so kernel. Activations are torch.float32 (Act::F32) or torch.bfloat16 (Act::BF16, raw bits).
"""
import ctypes
import functools
import struct

import torch

from . import (ACT_BF16, ACT_F32, GATE_NONE, GATE_SIGMOID, GATE_SILU, KV_BF16, KV_E4M3, MOE_F32, SCORE_SIGMOID, SCORE_SOFTMAX, SX_EINVAL, Fp8View,
               Int8View, LogitCand, MtpPick, QView, SxError, check, lib)

_c = ctypes.c_void_p


def _p(t):
    return None if t is None else _c(t.data_ptr())


def _s(stream=None):
    return _c((stream if stream is not None else torch.cuda.current_stream()).cuda_stream)


def act_of(t):
    if t.dtype == torch.float32:
        return ACT_F32
    if t.dtype == torch.bfloat16:
        return ACT_BF16
    raise TypeError(f"activations are float32 or bfloat16, got {t.dtype}")


def dtype_of(act):
    return torch.float32 if act == ACT_F32 else torch.bfloat16


def _empty(like, shape, dtype, stream, fill=None):
    """A buffer that a call makes, on like's device, from the pool of the stream that the call runs on (and filled there):
    from another one it could be memory that work queued there still uses, and if it is dropped, be given to such work
    while the call's kernels still write it."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _empty(like, shape, dtype, None, fill)
    t = like.new_empty(shape, dtype=dtype)
    return t if fill is None else t.fill_(fill)


def _empty_like(like, stream):
    """_empty in like's own shape and type (half of the host time)."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return torch.empty_like(like)
    return torch.empty_like(like)


class QWeight:
    """A q4 / q8 weight resident on the device (Q4Device / Q8Device, runtime/q4_device.hpp:23-36): codes uint8,
    scale / min as BF16 bits (int16 tensors), in the formats/q4.hpp / q8.hpp layout."""

    def __init__(self, bits, q, scale, minv, N, K, G):
        self.bits, self.q, self.scale, self.minv = bits, q, scale, minv
        self.N, self.K, self.G = int(N), int(K), int(G)
        self._view = QView(q.data_ptr(), scale.data_ptr(), minv.data_ptr(), self.N, self.K, self.G)

    @classmethod
    def upload(cls, host, device="cuda"):
        """From a host weight with numpy arrays q, scale, minv (e.g. oracle.QWeight)."""
        t = lambda a: torch.from_numpy(a.view(a.dtype)).to(device)
        return cls(host.bits, t(host.q), t(host.scale.view("int16")), t(host.minv.view("int16")), host.N, host.K, host.G)

    def view(self):
        return ctypes.byref(self._view)

    def nbytes(self):
        return self.q.numel() + 2 * self.scale.numel() + 2 * self.minv.numel()


def linear(x, w, out_act=None, y=None, stream=None):
    """y[M, N] = x[M, K] * deq(W)^T (linear_q4 / linear_q8)."""
    act = act_of(x)
    out_act = act if out_act is None else out_act
    M = x.shape[0]
    if y is None:
        y = _empty(x, (M, w.N), dtype_of(out_act), stream)
    f = lib().sx_linear_q4 if w.bits == 4 else lib().sx_linear_q8
    check(f(_p(x), w.view(), _p(y), M, act, out_act, _s(stream)))
    return y


def linear_kernel(w, M, act=ACT_BF16, out_act=None):
    """The kernel linear() runs for M rows of x against w: "k_split", "register_tiles", "wide_tiles_k_split",
    "wide_tiles" or "qmm"."""
    name = lib().sx_linear_kernel(w.view(), w.bits, M, act, act if out_act is None else out_act, 0)
    if name is None:
        raise SxError(SX_EINVAL, lib().sx_last_error().decode())
    return name.decode()


def experts_grouped_kernel(w, E, M, A, act=ACT_BF16):
    """The kernel gather_grouped() and combine_grouped() run: "register_tiles", "wide_tiles" or "qmm"."""
    name = lib().sx_experts_grouped_kernel(w.view(), E, M, A, act, 0)
    if name is None:
        raise SxError(SX_EINVAL, lib().sx_last_error().decode())
    return name.decode()


def _err(like, stream):
    """Zeroed error words for a call, on the call's stream (_empty)."""
    return _empty(like, (4,), torch.int32, stream, 0)


def experts_gather(x, w, E, ids, swiglu=False, y=None, err=None, stream=None):
    """Per-slot gather (linear_q4_experts_gather) or its SwiGLU form (linear_q4_experts_gather_swiglu)."""
    act = act_of(x)
    M, A = ids.shape
    N = w.N // E
    out_n = N // 2 if swiglu else N
    y = _empty(x, (M, A, out_n), x.dtype, stream) if y is None else y
    err = _err(x, stream) if err is None else err
    f = lib().sx_linear_q4_experts_gather_swiglu if swiglu else lib().sx_linear_q4_experts_gather
    check(f(_p(x), w.view(), E, _p(ids), M, A, _p(y), act, _p(err), _s(stream)))
    return y, err


def experts_combine(h, w, E, ids, coef, y=None, err=None, stream=None):
    act = act_of(h)
    M, A = ids.shape
    N = w.N // E
    y = _empty(h, (M, N), h.dtype, stream) if y is None else y
    err = _err(h, stream) if err is None else err
    check(lib().sx_linear_q4_experts_combine(_p(h), w.view(), E, _p(ids), _p(coef), M, A, _p(y), act, _p(err),
                                             _s(stream)))
    return y, err


def moe_router(logits, E, k, shared=None, shared_ld=1, shared_id=0, ids=None, coef=None, err=None, stream=None):
    M, ld = logits.shape
    A = k + (1 if shared is not None else 0)
    ids = _empty(logits, (M, A), torch.int32, stream) if ids is None else ids
    coef = _empty(logits, (M, A), torch.float32, stream) if coef is None else coef
    err = _err(logits, stream) if err is None else err
    check(lib().sx_moe_router(_p(logits), ld, M, E, k, _p(shared), shared_ld, shared_id, _p(ids), _p(coef),
                              act_of(logits), _p(err), _s(stream)))
    return ids, coef, err


def route_workspace_bytes(M, A, E):
    n = ctypes.c_size_t()
    check(lib().sx_moe_route_workspace_bytes(M, A, E, ctypes.byref(n)))
    return n.value


def router_group(logits, E, k, ws=None, ids=None, coef=None, router_err=None, expert_err=None, stream=None):
    """moe_router + moe_group_routes in one launch (M * k <= 2048)."""
    M, ld = logits.shape
    ws = _empty(logits, (route_workspace_bytes(M, k, E) // 4,), torch.int32, stream) if ws is None else ws
    ids = _empty(logits, (M, k), torch.int32, stream) if ids is None else ids
    coef = _empty(logits, (M, k), torch.float32, stream) if coef is None else coef
    router_err = _err(logits, stream) if router_err is None else router_err
    expert_err = _err(logits, stream) if expert_err is None else expert_err
    check(lib().sx_moe_router_group(_p(logits), ld, M, E, k, act_of(logits), _p(ids), _p(coef), _p(router_err),
                                    _p(ws), ws.numel() * 4, _p(expert_err), _s(stream)))
    return ids, coef, ws, router_err, expert_err


def verify_supported(M, A, E, k, Ew, gate_up, down, act=ACT_BF16):
    """Whether the two-launch verify FFN (verify_gate_up + verify_down) takes this shape."""
    return lib().sx_moe_verify_supported(M, A, E, k, Ew, gate_up.view(), down.view(), act) == 0


def verify_gate_up(x, logits, w, E, k, Ew=None, shared_logit=None, shared_id=0, ids=None, coef=None, h=None,
                   router_err=None, expert_err=None, h_sums=None, sync=None, plan=None, stream=None):
    """moe_router + gather_swiglu in one launch at verify width: ids, coef [M, A], h [M, A, I]. h_sums (optional,
    FP32 [M * A, ceil(I / 16)]) receives the 16-feature sums of h that verify_down can take. sync (optional,
    verify_layer_sync(), one per stream): after a fixed run each compute unit takes weight tiles from a shared pool
    (K = 4096), so the faster ones take more; same outputs. plan (optional, verify_plan()) receives the routing in
    the form verify_down takes it."""
    M, ld = x.shape[0], logits.stride(0)
    Ew = E if Ew is None else Ew
    A = k + (shared_logit is not None)
    I = w.N // Ew // 2
    ids = _empty(x, (M, A), torch.int32, stream) if ids is None else ids
    coef = _empty(x, (M, A), torch.float32, stream) if coef is None else coef
    h = _empty(x, (M, A, I), x.dtype, stream) if h is None else h
    router_err = _err(x, stream) if router_err is None else router_err
    expert_err = _err(x, stream) if expert_err is None else expert_err
    sld = 0 if shared_logit is None else shared_logit.stride(0)
    check(lib().sx_moe_verify_gate_up(_p(x), M, _p(logits), ld, E, k, _p(shared_logit), sld, shared_id, w.view(), Ew,
                                      _p(ids), _p(coef), _p(h), _p(h_sums), act_of(x), _p(router_err),
                                      _p(expert_err), _p(sync), _p(plan), _s(stream)))
    return ids, coef, h, router_err, expert_err


def verify_down(h, w, ids, coef, Ew, y=None, expert_err=None, h_sums=None, plan=None, stream=None):
    """y[M, N] = sum_a coef[m, a] * (h[m, a] . W[ids[m, a]]) in one launch at verify width (h_sums: verify_gate_up's
    sums of this h, optional; plan: the routing plan verify_gate_up stored with these ids, optional)."""
    M, A = ids.shape
    N = w.N // Ew
    y = _empty(h, (M, N), h.dtype, stream) if y is None else y
    expert_err = _err(h, stream) if expert_err is None else expert_err
    check(lib().sx_moe_verify_down(_p(h), _p(h_sums), M, A, _p(ids), _p(coef), w.view(), Ew, _p(y), act_of(h),
                                   _p(expert_err), _p(plan), _s(stream)))
    return y, expert_err


VERIFY_PLAN_BYTES = 4096  # SX_VERIFY_PLAN_BYTES


def verify_plan(device="cuda"):
    """A buffer for the routing plan verify_gate_up stores and verify_down takes."""
    return torch.empty(VERIFY_PLAN_BYTES // 4, dtype=torch.int32, device=device)


def verify_layer_sync(device="cuda"):
    """A zeroed sync buffer for verify_layer and verify_gate_up (one per stream; each launch readies it for the next)."""
    n = ctypes.c_size_t()
    check(lib().sx_moe_verify_layer_sync_bytes(ctypes.byref(n)))
    return torch.zeros((n.value + 3) // 4, dtype=torch.int32, device=device)


def verify_layer(x, Wr, gate_up, down, E, k, sync, shared=False, shared_id=0, Ew=None, logits=None, ids=None,
                 coef=None, h=None, h_sums=None, y=None, router_err=None, expert_err=None, stream=None):
    """The verify-width MoE sublayer in one launch: x [M, d] BF16, Wr [rows, d] FP32 or BF16 (raw bits as int16 or
    torch.bfloat16) -> logits [M, rows], ids / coef [M, A], h [M, A, I], h_sums, y [M, d]."""
    M, d = x.shape
    rows = Wr.shape[0]
    Ew = E if Ew is None else Ew
    A = k + (1 if shared else 0)
    I = gate_up.N // Ew // 2
    wr_act = ACT_F32 if Wr.dtype == torch.float32 else ACT_BF16
    logits = _empty(x, (M, rows), torch.float32, stream) if logits is None else logits
    ids = _empty(x, (M, A), torch.int32, stream) if ids is None else ids
    coef = _empty(x, (M, A), torch.float32, stream) if coef is None else coef
    h = _empty(x, (M, A, I), x.dtype, stream) if h is None else h
    h_sums = _empty(x, (M * A, (I + 15) // 16), torch.float32, stream) if h_sums is None else h_sums
    y = _empty(x, (M, down.N // Ew), x.dtype, stream) if y is None else y
    router_err = _err(x, stream) if router_err is None else router_err
    expert_err = _err(x, stream) if expert_err is None else expert_err
    check(lib().sx_moe_verify_layer(_p(x), M, _p(Wr), wr_act, rows, E, k, int(shared), shared_id, gate_up.view(),
                                    down.view(), Ew, _p(logits), _p(ids), _p(coef), _p(h), _p(h_sums), _p(y),
                                    act_of(x), _p(router_err), _p(expert_err), _p(sync), _s(stream)))
    return logits, ids, coef, h, y, router_err, expert_err


def group_routes(ids, E, ws=None, err=None, stream=None):
    M, A = ids.shape
    nb = route_workspace_bytes(M, A, E)
    ws = _empty(ids, (nb // 4,), torch.int32, stream) if ws is None else ws
    err = _err(ids, stream) if err is None else err
    check(lib().sx_moe_group_routes(_p(ids), M, A, E, _p(ws), ws.numel() * 4, _p(err), _s(stream)))
    return ws, err


def gather_grouped(x, w, E, ws, M, A, swiglu=False, y=None, math=MOE_F32, stream=None):
    act = act_of(x)
    N = w.N // E
    out_n = N // 2 if swiglu else N
    y = _empty(x, (M, A, out_n), x.dtype, stream) if y is None else y
    if swiglu:
        check(lib().sx_linear_q4_experts_gather_swiglu_grouped(_p(x), w.view(), E, _p(ws), ws.numel() * 4, M, A, _p(y),
                                                               act, _s(stream)))
    else:
        check(lib().sx_linear_q4_experts_gather_grouped(_p(x), w.view(), E, _p(ws), ws.numel() * 4, M, A, _p(y), act,
                                                        math, _s(stream)))
    return y


def combine_grouped(h, w, E, ids, coef, ws, partial=None, y=None, math=MOE_F32, stream=None):
    act = act_of(h)
    M, A = ids.shape
    N = w.N // E
    y = _empty(h, (M, N), h.dtype, stream) if y is None else y
    partial = _empty(h, (M * A, N), torch.float32, stream) if partial is None else partial
    check(lib().sx_linear_q4_experts_combine_grouped(_p(h), w.view(), E, _p(ids), _p(coef), _p(ws), ws.numel() * 4,
                                                     _p(partial), M, A, _p(y), act, math, _s(stream)))
    return y


def swiglu(gu, h=None, stream=None):
    rows, I2 = gu.shape
    h = _empty(gu, (rows, I2 // 2), gu.dtype, stream) if h is None else h
    check(lib().sx_swiglu(_p(gu), _p(h), rows, I2 // 2, act_of(gu), _s(stream)))
    return h


def linear_f32w(x, W, y=None, stream=None):
    M, K = x.shape
    N = W.shape[0]
    y = _empty(x, (M, N), torch.float32, stream) if y is None else y
    check(lib().sx_linear_f32w(_p(x), _p(W), N, K, _p(y), M, act_of(x), _s(stream)))
    return y


def linear_bf16w(x, W, out_act=None, y=None, wmma=False, stream=None):
    """y[M, N] = x[M, K] * W^T with W BF16 [N, K] (linear_bf16w; wmma: linear_bf16w_wmma, x rounded to BF16)."""
    act = act_of(x)
    out_act = act if out_act is None else out_act
    M, K = x.shape
    N = W.shape[0]
    y = _empty(x, (M, N), dtype_of(out_act), stream) if y is None else y
    f = lib().sx_linear_bf16w_wmma if wmma else lib().sx_linear_bf16w
    check(f(_p(x), _p(W), _p(y), M, N, K, act, out_act, _s(stream)))
    return y


def moe_shared_add(y, s, gate_logit, gate_index, err, x=None, w_in=None, stream=None):
    """moe_shared_add (x None) or moe_shared_add_inject, in place on y (and x [M, H * N]). gate_logit: FP32 column
    view (row stride = its stride(0))."""
    M, N = y.shape
    gl = gate_logit.stride(0)
    if x is None:
        check(lib().sx_moe_shared_add(_p(y), _p(s), _p(gate_logit), gl, M, N, gate_index, act_of(y), _p(err),
                                      _s(stream)))
    else:
        check(lib().sx_moe_shared_add_inject(_p(y), _p(s), _p(gate_logit), gl, M, N, gate_index, _p(x), _p(w_in),
                                             x.shape[1] // N, act_of(y), _p(err), _s(stream)))
    return y


def topk_workspace_bytes(rows, n_valid, k):
    n = ctypes.c_size_t()
    check(lib().sx_logits_topk_workspace_bytes(rows, n_valid, k, ctypes.byref(n)))
    return n.value


def logits_topk(logits, n_valid, k=20, mask=None, ws=None, out=None, nan=None, stream=None):
    """Per row the best k (value desc, lower id on a tie) of logits [rows, >= n_valid] (any row stride). Returns
    (values f32 [rows, k], ids i32 [rows, k], nan, the raw [rows, k, 2] candidates)."""
    rows, ld = logits.shape[0], logits.stride(0)
    out = _empty(logits, (rows, k, 2), torch.int32, stream) if out is None else out
    nan = _empty(logits, (rows,), torch.int32, stream) if nan is None else nan
    if ws is None:
        ws = _empty(logits, (topk_workspace_bytes(rows, n_valid, k) // 8 + 1,), torch.int64, stream)
    mw = 0 if mask is None else mask.shape[1]
    check(lib().sx_logits_topk(_p(logits), rows, ld, n_valid, k, _p(out), _p(nan), _p(ws), ws.numel() * 8, _p(mask), mw,
                               _s(stream)))
    return out[..., 0].view(torch.float32), out[..., 1], nan, out


def logits_topk_noalloc(logits, n_valid, k=20, mask=None, out=None, nan=None, stream=None):
    """logits_topk on the library's fixed scratch (sx_logits_topk_noalloc: no workspace, nothing allocated by the
    call). Same returns as logits_topk."""
    rows, ld = logits.shape[0], logits.stride(0)
    out = _empty(logits, (rows, k, 2), torch.int32, stream) if out is None else out
    nan = _empty(logits, (rows,), torch.int32, stream) if nan is None else nan
    mw = 0 if mask is None else mask.shape[1]
    check(lib().sx_logits_topk_noalloc(_p(logits), rows, ld, n_valid, k, _p(out), _p(nan), _p(mask), mw, _s(stream)))
    return out[..., 0].view(torch.float32), out[..., 1], nan, out


def quantize_q4_from_q8(w8, G=64, rows=None, err=None, stream=None):
    """The Q4 copy of the first `rows` rows of a Q8 weight (formats/q4_from_q8.hpp), made on the device: a QWeight."""
    rows = w8.N if rows is None else rows
    q = _empty(w8.q, (rows * w8.K // 2,), torch.uint8, stream)
    s = _empty(w8.q, (rows * (w8.K // G),), torch.int16, stream)
    m = _empty(w8.q, (rows * (w8.K // G),), torch.int16, stream)
    err = _err(w8.q, stream) if err is None else err
    src = QView(w8.q.data_ptr(), w8.scale.data_ptr(), w8.minv.data_ptr(), rows, w8.K, w8.G)
    check(lib().sx_quantize_q4_from_q8(ctypes.byref(src), G, _p(q), _p(s), _p(m), _p(err), _s(stream)))
    return QWeight(4, q, s, m, rows, w8.K, G), err


def mtp_pick_ws_bytes(n):
    b = ctypes.c_size_t()
    check(lib().sx_mtp_pick_ws_bytes(n, ctypes.byref(b)))
    return b.value


def mtp_pick(logits, router_err, expert_err, attn_err, emb_err, out=None, ws=None, stream=None):
    """The 64-byte pick of `logits`. With `ws` (a zeroed device uint8 buffer of mtp_pick_ws_bytes, reused across
    calls on one stream) the one-launch many-block pick runs; its output is bit-identical to the single-block one's."""
    out = _empty(logits, (64,), torch.uint8, stream) if out is None else out
    if ws is None:
        check(lib().sx_mtp_pick(_p(logits), logits.numel(), _p(router_err), _p(expert_err), _p(attn_err),
                                _p(emb_err), _p(out), _s(stream)))
    else:
        check(lib().sx_mtp_pick_ws(_p(logits), logits.numel(), _p(router_err), _p(expert_err), _p(attn_err),
                                   _p(emb_err), _p(out), _p(ws), ws.numel() * ws.element_size(), _s(stream)))
    return out


def mtp_head_pick(x, w, logits, router_err, expert_err, attn_err, emb_err, ws, out=None, stream=None):
    """The draft head's logits (x BF16 [1, K] against the q4 / q8 head, FP32 [N] into `logits`) and their pick, one
    launch; `ws` a zeroed device uint8 buffer of mtp_pick_ws_bytes. Returns the 64-byte pick."""
    out = _empty(x, (64,), torch.uint8, stream) if out is None else out
    assert x.dtype == torch.bfloat16 and x.numel() == w.K and logits.numel() >= w.N
    check(lib().sx_mtp_head_pick(_p(x), w.view(), w.bits, _p(logits), _p(router_err), _p(expert_err), _p(attn_err),
                                 _p(emb_err), _p(out), _p(ws), ws.numel() * ws.element_size(), _s(stream)))
    return out


def pick_from_bytes(b):
    """The 64 bytes of an sx_mtp_pick_t (host) as the ctypes struct."""
    return MtpPick.from_buffer_copy(bytes(b.cpu().numpy().tobytes()))


def verify_tail_workspace_bytes(rows, n_valid, kc):
    n = ctypes.c_size_t()
    check(lib().sx_verify_tail_workspace_bytes(rows, n_valid, kc, ctypes.byref(n)))
    return n.value


def verify_tail_workspace(rows, n_valid, kc, device="cuda"):
    """A zeroed workspace for verify_tail (one per stream; each launch leaves its counters at zero)."""
    return torch.zeros(verify_tail_workspace_bytes(rows, n_valid, kc) // 8 + 1, dtype=torch.int64, device=device)


def verify_tail(logits, n_valid, kc, ws, drafts=None, u=None, temperature=0.0, top_k=1, top_p=1.0, mask=None,
                cands=None, nan=None, out=None, stream=None):
    """logits_topk (kc candidates a row) and, with drafts, mtp_accept in one launch. Returns (cands [rows, kc, 2],
    nan, out or None)."""
    rows, ld = logits.shape[0], logits.stride(0)
    cands = _empty(logits, (rows, kc, 2), torch.int32, stream) if cands is None else cands
    nan = _empty(logits, (rows,), torch.int32, stream) if nan is None else nan
    k = 0 if drafts is None else drafts.numel()
    if drafts is not None and out is None:
        out = _empty(logits, (2 + k + 1,), torch.int32, stream, -1)
    mw = 0 if mask is None else mask.shape[1]
    check(lib().sx_verify_tail(_p(logits), rows, ld, n_valid, kc, _p(cands), _p(nan), _p(mask), mw, _p(drafts), k,
                               _p(u), float(temperature), int(top_k), float(top_p),
                               _p(out) if drafts is not None else None, _p(ws), ws.numel() * 8, _s(stream)))
    return cands, nan, out


def mtp_accept(cands, nan, drafts, u, temperature, top_k, top_p, n_valid, out=None, stream=None):
    """cands: the raw [k+1, kc, 2] int32 output of logits_topk. Returns the device int32 vector
    [j, status, tokens...]."""
    rows, kc = cands.shape[0], cands.shape[1]
    k = drafts.numel()
    assert rows >= k + 1, "one candidate row per draft plus the last"
    out = _empty(cands, (2 + k + 1,), torch.int32, stream, -1) if out is None else out
    check(lib().sx_mtp_accept(_p(cands), _p(nan), kc, _p(drafts), k, _p(u), float(temperature), int(top_k),
                              float(top_p), int(n_valid), _p(out), _s(stream)))
    return out


# ---------------- a verify layer's attention half, and routing by scores ----------------
# Strides, types, shapes and devices are checked here, where the tensors are; the library checks the rest. A call runs
# on its tensors' device, on that device's current stream unless one is given; buffers that it makes come from that
# stream's pool. err (optional, a zeroed int32 [4] on the device) receives what a call could not read; without it the
# outputs alone say so.

def _refuse(*what):
    raise SxError(SX_EINVAL, " ".join(str(w) for w in what))


def _is(name, t, dtype, shape):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        _refuse(name, "must be a contiguous", dtype, tuple(shape), "and is", t.dtype, tuple(t.shape), t.stride())


def _together(dev, tensors):
    """Refuses tensors (None: left out) that are not on GPU `dev`, a tensor's get_device()."""
    if dev < 0:
        _refuse("the tensors are not on a GPU")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _refuse("tensors on", t.device, "and on GPU", dev, "in one call")


def _is_err(err):
    if err is not None and (err.dtype != torch.int32 or err.numel() < 4 or not err.is_contiguous()):
        _refuse("err must be a contiguous int32 [4] and is", err.dtype, tuple(err.shape), err.stride())


def _run(dev, f, *args, stream=None):
    """f(*args, stream) on GPU dev, whichever is current."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _run(dev, f, *args, stream=stream)
    rc = f(*args, torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream)
    if rc:
        check(rc)


def _a(t):
    return None if t is None else t.data_ptr()


class Fp8Weight:
    """An e4m3 weight resident on the device: q [N, K] torch.float8_e4m3fn, scale [ceil(N / 128), K / 128] FP32, one
    for each 128 x 128 tile (w = code * scale)."""

    def __init__(self, q, scale):
        if q.dim() != 2 or q.shape[1] % 128:
            _refuse("an FP8 weight is [N, K], K a multiple of 128, and not", tuple(q.shape))
        self.N, self.K = (int(n) for n in q.shape)
        _is("q", q, torch.float8_e4m3fn, (self.N, self.K))
        _is("scale", scale, torch.float32, (-(-self.N // 128), self.K // 128))
        if scale.device != q.device:
            _refuse("q is on", q.device, "and scale on", scale.device)
        self.q, self.scale = q, scale
        self._view = Fp8View(q.data_ptr(), scale.data_ptr(), self.N, self.K)

    def view(self):
        return ctypes.byref(self._view)

    def nbytes(self):
        return self.q.numel() + 4 * self.scale.numel()


def add_rms_norm_fp8(x, weight, eps=1e-6, residual=None, residual_out=None, w_add=0.0, y=None, q=None, scale=None,
                     stream=None):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * (weight + w_add) as e4m3 codes q [M, K] and FP32 scales
    [M, K / 128], the activations linear_fp8 takes. x [M, K] (any row stride) in FP32 or BF16; y (optional): a buffer
    that receives y itself in x's type. Returns (q, scale, residual_out or None); residual_out may be the residual."""
    act, dtype, dev = act_of(x), x.dtype, x.get_device()
    if x.dim() != 2 or x.stride(1) != 1 or x.shape[1] % 128:
        _refuse("x must be [M, K] with dense rows, K a multiple of 128, and is", tuple(x.shape), x.stride())
    M, K = shape = x.shape
    _together(dev, (weight, residual, residual_out, y, q, scale))
    _is("weight", weight, dtype, (K,))
    if residual is not None:
        _is("residual", residual, dtype, shape)
        if residual_out is None:
            residual_out = _empty_like(residual, stream)
        else:
            _is("residual_out", residual_out, dtype, shape)
    elif residual_out is not None:
        _refuse("residual_out without a residual")
    if y is not None:
        _is("y", y, dtype, shape)
    if q is None:
        q = _empty(x, shape, torch.float8_e4m3fn, stream)
    else:
        _is("q", q, torch.float8_e4m3fn, shape)
    if scale is None:
        scale = _empty(x, (M, K // 128), torch.float32, stream)
    else:
        _is("scale", scale, torch.float32, (M, K // 128))
    _run(dev, lib().sx_add_rms_norm_fp8, x.data_ptr(), x.stride(0) if M > 1 else K, _a(residual), weight.data_ptr(), M, K,
         eps, w_add, _a(residual_out), _a(y), q.data_ptr(), scale.data_ptr(), act, stream=stream)
    return q, scale, residual_out


def linear_fp8(x, x_scale, w, out_act=ACT_BF16, y=None, stream=None):
    """y[M, N] = (x * x_scale) * w^T: x e4m3 codes [M, K] with an FP32 scale for each run of 128 (add_rms_norm_fp8's
    outputs), w an Fp8Weight; y BF16 or (out_act ACT_F32) FP32."""
    dev, M, dtype = x.get_device(), x.shape[0], dtype_of(out_act)
    _together(dev, (x_scale, w.q, y))
    _is("x", x, torch.float8_e4m3fn, (M, w.K))
    _is("x_scale", x_scale, torch.float32, (M, w.K // 128))
    if y is None:
        y = _empty(x, (M, w.N), dtype, stream)
    else:
        _is("y", y, dtype, (M, w.N))
    _run(dev, lib().sx_linear_fp8, x.data_ptr(), x_scale.data_ptr(), w.view(), y.data_ptr(), M, out_act, stream=stream)
    return y


# sx_head_rows and sx_kv_cache as bytes: a quarter of the host time of building the ctypes structures
_ROWS, _CACHE = struct.Struct("@P3q").pack, struct.Struct("@2Pi2f5q8qP2qPq").pack


def _head_rows(name, t, heads, dim, layered=False):
    """The sx_head_rows of a BF16 tensor [T, heads, dim] (layered: [layers, T, heads, dim]); dims dense, other strides
    free."""
    if t.dtype != torch.bfloat16 or t.dim() != 3 + layered or t.shape[-2:] != (heads, dim) or t.stride(-1) != 1:
        _refuse(name, f"must be BF16 [tokens, {heads}, {dim}] with dense rows and is", t.dtype, tuple(t.shape), t.stride())
    s = t.stride()
    return _ROWS(t.data_ptr(), s[-3], s[-2], s[0] if layered else 0)


def _kv_cache(k, v, table, lens, k_scale, v_scale, layered=False):
    """The sx_kv_cache of [pages, page, heads, dim] tensors (layered: [layers, ...]) with free strides, and (sequences,
    heads, dim, layers)."""
    dtype = k.dtype
    if dtype != torch.bfloat16 and dtype != torch.float8_e4m3fn or v.dtype != dtype:
        _refuse("the cache is BF16 or float8_e4m3fn, not", dtype, v.dtype)
    ks, vs, shape = k.stride(), v.stride(), k.shape
    if len(shape) != 4 + layered or v.shape != shape or ks[-1] != 1 or vs[-1] != 1:
        _refuse("k and v caches must be [pages, page, heads, dim] alike with dense rows:", tuple(shape), tuple(v.shape))
    if table.dtype != torch.int32 or table.dim() != 2 or table.stride(1) != 1:
        _refuse("table must be int32 [batch, pages a sequence] with dense rows")
    B, P = table.shape
    _is("lens", lens, torch.int32, (B,))
    pages, page, heads, dim = shape[-4:]
    layers = shape[0] if layered else 1
    c = _CACHE(k.data_ptr(), v.data_ptr(), KV_BF16 if dtype == torch.bfloat16 else KV_E4M3, k_scale, v_scale, pages, page,
               heads, dim, layers, ks[-4], ks[-3], ks[-2], ks[0] if layered else 0, vs[-4], vs[-3], vs[-2],
               vs[0] if layered else 0, table.data_ptr(), table.stride(0) if B > 1 else P, P, lens.data_ptr(), B)
    return c, (B, heads, dim, layers)


def tree_mask(parents):
    """The mask of drafted trees: parents is one list a sequence, each token's parent in it (-1: a root, which sees the
    cache alone; a parent comes before its children). Returns int64 [T, ceil(longest / 64)] on the host: bit j of a
    token's words says that it sees drafted token j of its sequence, itself and its ancestors."""
    words = (max((len(p) for p in parents), default=0) + 63) // 64
    rows = []
    for seq in parents:
        first = len(rows)
        for i, p in enumerate(seq):
            if not -1 <= p < i:
                raise ValueError(f"token {i} has parent {p}")
            rows.append((rows[first + p] if p >= 0 else 0) | 1 << i)
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    return torch.tensor([[signed(r >> 64 * i & (1 << 64) - 1) for i in range(words)] for r in rows], dtype=torch.int64)


def tree_attention_workspace_bytes(B, Hq, Hkv, D, max_new):
    n = ctypes.c_size_t()
    check(lib().sx_tree_attention_workspace_bytes(B, Hq, Hkv, D, max_new, ctypes.byref(n)))
    return n.value


def tree_attention_workspace(q, k_new, starts, max_new):
    """A workspace for tree_attention calls of these shapes (one per stream; nothing in it outlives a call)."""
    with torch.cuda.device(q.device):
        n = tree_attention_workspace_bytes(starts.numel() - 1, q.shape[1], k_new.shape[1], q.shape[2], max_new)
    return torch.empty((n + 7) // 8, dtype=torch.int64, device=q.device)


def tree_attention(q, k_new, v_new, k_cache, v_cache, table, lens, starts, mask, max_new, scale=None, k_scale=1.0,
                   v_scale=1.0, out=None, lse=None, ws=None, err=None, stream=None):
    """Attention of drafted tokens (q [T, Hq, D], k_new and v_new [T, Hkv, D], BF16, any token and head strides) over
    their sequences' cached tokens and, as the mask says, each other. The cache: k_cache, v_cache [pages, page, Hkv, D]
    (BF16, or float8_e4m3fn holding value / k_scale and value / v_scale), table int32 [B, pages a sequence], lens int32
    [B]. starts int32 [B + 1]: sequence b's drafted tokens are rows starts[b] .. starts[b + 1] - 1, at most max_new.
    mask int64 [T, words] as tree_mask makes it. scale: of the scores, 1 / sqrt(D) unless given. lse (optional): an
    FP32 [T, Hq] buffer for the rows' log sums. ws: tree_attention_workspace(), made for the call unless given. Returns
    (out [T, Hq, D] BF16, err)."""
    dev = q.get_device()
    if q.dim() != 3 or k_new.dim() != 3:
        _refuse("q, k_new and v_new are [tokens, heads, dim]")
    T, Hq, D = q.shape
    Hkv = k_new.shape[1]
    _together(dev, (k_new, v_new, k_cache, v_cache, table, lens, starts, mask, out, lse, ws, err))
    cache, (B, heads, dim, _) = _kv_cache(k_cache, v_cache, table, lens, k_scale, v_scale)
    if (heads, dim) != (Hkv, D) or k_new.shape[0] != T or v_new.shape[0] != T:
        _refuse("q", tuple(q.shape), "k_new", tuple(k_new.shape), "v_new", tuple(v_new.shape), "cache", tuple(k_cache.shape))
    _is("starts", starts, torch.int32, (B + 1,))
    if mask.dtype != torch.int64 or mask.dim() != 2 or mask.shape[0] != T or mask.stride(1) != 1 or mask.shape[1] * 64 < max_new:
        _refuse("mask must be int64 [T, ceil(max_new / 64)] with dense rows and is", mask.dtype, tuple(mask.shape))
    if out is None:
        out = _empty(q, (T, Hq, D), torch.bfloat16, stream)
    elif out.dim() != 3 or out.shape[0] != T:
        _refuse("out is", tuple(out.shape))
    if lse is not None:
        _is("lse", lse, torch.float32, (T, Hq))
    if ws is None:
        with torch.cuda.stream(stream):  # as _empty's (None: the current one's)
            ws = tree_attention_workspace(q, k_new, starts, max_new)
    elif not ws.is_contiguous():
        _refuse("ws must be contiguous and has strides", ws.stride())
    _is_err(err)
    rq, rk, rv = _head_rows("q", q, Hq, D), _head_rows("k_new", k_new, Hkv, D), _head_rows("v_new", v_new, Hkv, D)
    _run(dev, lib().sx_tree_attention, rq, rk, rv, T, Hq, cache, starts.data_ptr(), max_new, mask.data_ptr(),
         mask.stride(0) if T > 1 else mask.shape[1], D ** -0.5 if scale is None else scale, _head_rows("out", out, Hq, D),
         _a(lse), ws.data_ptr(), ws.numel() * ws.element_size(), _a(err), stream=stream)
    return out, err


def kv_append(k_new, v_new, k_cache, v_cache, table, lens, starts, count, path=None, max_count=None, k_scale=1.0,
              v_scale=1.0, lens_out=None, err=None, stream=None):
    """The accepted drafted tokens into the paged cache, all layers in one launch: for i < count[b], row
    starts[b] + path[b, i] (path None: starts[b] + i) of k_new and v_new [layers, T, Hkv, D] to position lens[b] + i of
    k_cache and v_cache [layers, pages, page, Hkv, D] (one layer: without that dimension). count int32 [B]; path int32
    [B, at most], whose width bounds the counts (without a path max_count does). Returns (lens_out = lens + count,
    err); lens itself is only read. A sequence that cannot be appended to as asked keeps its length and its pages."""
    dev, layered, shape = k_new.get_device(), k_new.dim() == 4, k_new.shape
    if len(shape) not in (3, 4) or v_new.shape != shape:
        _refuse("k_new", tuple(shape), "and v_new", tuple(v_new.shape))
    _together(dev, (v_new, k_cache, v_cache, table, lens, starts, count, path, lens_out, err))
    cache, (B, heads, dim, layers) = _kv_cache(k_cache, v_cache, table, lens, k_scale, v_scale, layered)
    T = shape[-3]
    if layered and shape[0] != layers:
        _refuse("k_new has", shape[0], "layers and the cache", layers)
    rk, rv = _head_rows("k_new", k_new, heads, dim, layered), _head_rows("v_new", v_new, heads, dim, layered)
    _is("starts", starts, torch.int32, (B + 1,))
    _is("count", count, torch.int32, (B,))
    ld = 0
    if path is not None:
        if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != B or path.stride(1) != 1:
            _refuse("path must be int32 [batch, most tokens kept] with dense rows")
        max_count = path.shape[1] if max_count is None else max_count
        ld = path.stride(0) if B > 1 else path.shape[1]
        if max_count > path.shape[1]:
            _refuse("max_count =", max_count, "is over the path's", path.shape[1])
    elif max_count is None:
        _refuse("max_count is needed without a path")
    if lens_out is None:
        lens_out = _empty_like(lens, stream)
    else:
        _is("lens_out", lens_out, torch.int32, (B,))
    _is_err(err)
    _run(dev, lib().sx_kv_append, rk, rv, T, cache, starts.data_ptr(), count.data_ptr(), max_count, _a(path),
         ld, lens_out.data_ptr(), _a(err), stream=stream)
    return lens_out, err


SCORES = {"sigmoid": SCORE_SIGMOID, "softmax": SCORE_SOFTMAX}


def moe_router_scored(logits, E, k, score="sigmoid", bias=None, groups=1, top_groups=1, group_best=2, renorm=True,
                      factor=1.0, shared=None, shared_ld=1, shared_id=0, ids=None, coef=None, err=None, stream=None):
    """Routing by scores: s = sigmoid or softmax of logits [M, >= E] (any row stride); the k experts with the largest
    s + bias, inside the top_groups of `groups` runs of experts by the sum of their group_best best; coef = s of those,
    divided by their sum if renorm, times factor. bias FP32 [E] or None. The shared slot as moe_router's. Returns (ids,
    coef, err)."""
    dev, act = logits.get_device(), act_of(logits)
    if logits.dim() != 2 or logits.stride(1) != 1 or logits.shape[1] < E:
        _refuse("logits are", tuple(logits.shape), logits.stride(), "for E =", E)
    if score not in SCORES:
        _refuse("score is", repr(score), "and not one of", list(SCORES))
    M = logits.shape[0]
    shape = (M, k + (1 if shared is not None else 0))
    _together(dev, (bias, shared, ids, coef, err))
    if bias is not None:
        _is("bias", bias, torch.float32, (E,))
    if shared is not None and (shared.dtype != logits.dtype or shared.shape[0] != M):
        _refuse("shared is", shared.dtype, tuple(shared.shape), "for logits", logits.dtype, tuple(logits.shape))
    if shared is not None and (shared.storage_offset() + (M - 1) * shared_ld + 1) * shared.element_size() > shared.untyped_storage().nbytes():
        _refuse("shared_ld =", shared_ld, "leads past the shared logits", tuple(shared.shape), shared.stride())
    if ids is None:
        ids = _empty(logits, shape, torch.int32, stream)
    else:
        _is("ids", ids, torch.int32, shape)
    if coef is None:
        coef = _empty(logits, shape, torch.float32, stream)
    else:
        _is("coef", coef, torch.float32, shape)
    _is_err(err)
    _run(dev, lib().sx_moe_router_scored, logits.data_ptr(), logits.stride(0) if M > 1 else logits.shape[1], M, E, k,
         SCORES[score], _a(bias), groups, top_groups if groups > 1 else 1, group_best if groups > 1 else 1, int(renorm),
         factor, _a(shared), shared_ld, shared_id, ids.data_ptr(), coef.data_ptr(), act, _a(err), stream=stream)
    return ids, coef, err


# ---------------- 8-bit integer activations and linear ----------------

GATES = {"none": GATE_NONE, "silu": GATE_SILU, "sigmoid": GATE_SIGMOID}
_NORM = struct.Struct("@9P4qi4d").pack  # sx_block_norm as bytes


def block_norm_int8(x, post=None, gate=None, residual=None, pre=None, eps=1e-6, w_add=0.0, group=None, gate_act="none",
                    residual_scale=1.0, branch_scale=1.0, residual_out=None, y=None, q=None, scale=None, codes=True, stream=None):
    """h = x / rms(x) * (post + w_add), over the row or each run of `group` features; h *= act(gate), act none, silu or sigmoid;
    r = residual_scale * residual + branch_scale * h (with a residual: rounded, residual_out); y = r / rms(r) * (pre + w_add); and y as
    int8 codes q [M, K] with an FP32 scale for each row [M], the activations linear_int8 takes. Each of post, gate, residual and pre
    may be None and is then left out. x [M, K] (any row stride) in FP32 or BF16, the others in its type: gate [M, K], its rows any
    stride apart (expanded: one for all), post [K] or [group], pre [K], y (optional): a buffer that receives y itself. codes False: no
    q and scale. Returns (q, scale, residual_out or None); residual_out may be the residual."""
    act, dtype, dev = act_of(x), x.dtype, x.get_device()
    shape, xt = x.shape, x.stride()
    if len(shape) != 2 or xt[1] != 1:
        _refuse("x must be [M, K] with dense rows and is", tuple(shape), xt)
    M, K = shape
    _together(dev, (post, gate, residual, pre, residual_out, y, q, scale))
    post_len, ldg = 0, 0
    if post is not None:
        post_len = post.shape[0]
        if post.dtype is not dtype or post.dim() != 1 or post_len != K and post_len != group or not post.is_contiguous():
            _is("post", post, dtype, (K,))
    if gate is not None:
        ldg, g1 = gate.stride() if gate.dim() == 2 else (0, 0)
        if gate.dtype is not dtype or gate.shape != shape or g1 != 1:
            _refuse("gate must be", dtype, tuple(shape), "with dense rows and is", gate.dtype, tuple(gate.shape), gate.stride())
    if gate_act not in GATES:
        _refuse("gate_act is", repr(gate_act), "and not one of", list(GATES))
    if pre is not None and (pre.dtype is not dtype or pre.shape != (K,) or not pre.is_contiguous()):
        _is("pre", pre, dtype, (K,))
    if residual is not None:
        if residual.dtype is not dtype or residual.shape != shape or not residual.is_contiguous():
            _is("residual", residual, dtype, shape)
        if residual_out is None:
            residual_out = _empty_like(residual, stream)
        elif residual_out.dtype is not dtype or residual_out.shape != shape or not residual_out.is_contiguous():
            _is("residual_out", residual_out, dtype, shape)
    elif residual_out is not None:
        _refuse("residual_out without a residual")
    if y is not None and (y.dtype is not dtype or y.shape != shape or not y.is_contiguous()):
        _is("y", y, dtype, shape)
    if not codes:
        if q is not None or scale is not None:
            _refuse("q or scale without codes")
    else:
        if q is None:
            q = _empty(x, shape, torch.int8, stream)
        else:
            _is("q", q, torch.int8, shape)
        if scale is None:
            scale = _empty(x, (M,), torch.float32, stream)
        else:
            _is("scale", scale, torch.float32, (M,))
    a = lambda t: 0 if t is None else t.data_ptr()
    n = _NORM(x.data_ptr(), a(post), a(gate), a(residual), a(pre), a(residual_out), a(y), a(q), a(scale), xt[0] if M > 1 else K,
              ldg if M > 1 else K, group or 0, post_len, GATES[gate_act], eps, w_add, residual_scale,
              branch_scale)
    _run(dev, lib().sx_block_norm_int8, n, M, K, act, stream=stream)
    return q, scale, residual_out



class Int8Weight:
    """An int8 weight resident on the device: q [N, K] torch.int8, scale [N] FP32, one for each channel (w = code * scale)."""

    def __init__(self, q, scale):
        if q.dim() != 2 or q.shape[1] % 16:
            _refuse("an int8 weight is [N, K], K a multiple of 16, and not", tuple(q.shape))
        self.N, self.K = (int(n) for n in q.shape)
        _is("q", q, torch.int8, (self.N, self.K))
        _is("scale", scale, torch.float32, (self.N,))
        if scale.device != q.device:
            _refuse("q is on", q.device, "and scale on", scale.device)
        self.q, self.scale = q, scale
        self._view = Int8View(q.data_ptr(), scale.data_ptr(), self.N, self.K)

    def view(self):
        return ctypes.byref(self._view)

    def nbytes(self):
        return self.q.numel() + 4 * self.scale.numel()


def linear_int8(x, x_scale, w, out_act=ACT_BF16, y=None, stream=None):
    """y[M, N] = (x * x_scale) * w^T: x int8 codes [M, K] with an FP32 scale for each token [M] (block_norm_int8's outputs), w an
    Int8Weight; y BF16 or (out_act ACT_F32) FP32."""
    dev, M, dtype = x.get_device(), x.shape[0], dtype_of(out_act)
    _together(dev, (x_scale, w.q, y))
    _is("x", x, torch.int8, (M, w.K))
    _is("x_scale", x_scale, torch.float32, (M,))
    if y is None:
        y = _empty(x, (M, w.N), dtype, stream)
    else:
        _is("y", y, dtype, (M, w.N))
    _run(dev, lib().sx_linear_int8, x.data_ptr(), x_scale.data_ptr(), w.view(), y.data_ptr(), M, out_act, stream=stream)
    return y


# ---------------- the gated delta rule ----------------

# sx_delta as bytes
_DELTA = struct.Struct("@Pqqq Pqqq Pqqq PP qq PPPPP qqqqqqqq iif4x".replace(" ", "")).pack


_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _delta_refuse(q, k, v, a, b, state, starts, slots, A_log, dt_bias):
    """What of these tensors is not as _delta needs it."""
    if q.dim() != 3 or v.dim() != 3:
        _refuse("q, k and v are [tokens, heads, dim]")
    (T, Hk, Dk), (Hv, Dv) = q.shape, v.shape[1:]
    if k.shape != q.shape or v.shape[0] != T:
        _refuse("q", tuple(q.shape), "k", tuple(k.shape), "v", tuple(v.shape))
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != _BF16 or t.stride(2) != 1:
            _refuse(name, "must be BF16 [tokens, heads, dim] with dense rows and is", t.dtype, tuple(t.shape), t.stride())
    for name, t in (("a", a), ("b", b)):
        if t.shape != (T, Hv) or t.stride(1) != 1 or t.dtype != a.dtype:
            _refuse(name, f"must be [{T}, {Hv}] with dense rows, a and b of one type, and is", t.dtype, tuple(t.shape), t.stride())
    if state.dtype != _F32 or state.dim() != 4 or state.shape[1:] != (Hv, Dk, Dv) or state.stride()[1:] != (Dk * Dv, Dv, 1):
        _refuse(f"state must be FP32 [states, {Hv}, {Dk}, {Dv}], each dense, and is", state.dtype, tuple(state.shape), state.stride())
    if starts.dim() != 1 or starts.numel() < 2:
        _refuse("starts must be [batch + 1] and is", tuple(starts.shape))
    B = starts.numel() - 1
    _is("starts", starts, _I32, (B + 1,))
    if slots is not None:
        _is("slots", slots, _I32, (B,))
    if A_log is not None:
        _is("A_log", A_log, _F32, (Hv,))
    if dt_bias is not None:
        _is("dt_bias", dt_bias, _F32, (Hv,))


def _delta(q, k, v, a, b, state, starts, slots, A_log, dt_bias, normalize, scale):
    """The sx_delta of these tensors, and (T, Hk, Hv, Dk, Dv, batch). All is looked at in one expression; what is wrong is found out
    only where something is (half of the host time)."""
    qs, vs, ss = q.shape, v.shape, state.shape
    if len(qs) != 3 or len(vs) != 3 or len(ss) != 4 or a.dim() != 2 or b.dim() != 2 or starts.dim() != 1:
        _delta_refuse(q, k, v, a, b, state, starts, slots, A_log, dt_bias)
        _refuse("a and b are [tokens, heads]")
    T, Hk, Dk = qs
    Tv, Hv, Dv = vs
    (qt, qh, q1), (kt, kh, k1), (vt, vh, v1) = q.stride(), k.stride(), v.stride()
    (at, a1), (bt, b1), (st, s1, s2, s3), (n, heads, dk, dv) = a.stride(), b.stride(), state.stride(), ss
    B, dtype, g = starts.shape[0] - 1, q.dtype, (T, Hv)
    if (k.shape != qs or Tv != T or dtype is not _BF16 or k.dtype is not dtype or v.dtype is not dtype or q1 * k1 * v1 * a1 * b1 * s3 != 1 or
            a.shape != g or b.shape != g or b.dtype is not a.dtype or state.dtype is not _F32 or heads != Hv or dk != Dk or dv != Dv or
            s1 != Dk * Dv or s2 != Dv or B < 1 or starts.dtype is not _I32 or not starts.is_contiguous() or
            slots is not None and (slots.dtype is not _I32 or slots.shape != (B,) or not slots.is_contiguous()) or
            A_log is not None and (A_log.dtype is not _F32 or A_log.shape != (Hv,) or not A_log.is_contiguous()) or
            dt_bias is not None and (dt_bias.dtype is not _F32 or dt_bias.shape != (Hv,) or not dt_bias.is_contiguous())):
        _delta_refuse(q, k, v, a, b, state, starts, slots, A_log, dt_bias)
    d = _DELTA(q.data_ptr(), qt, qh, 0, k.data_ptr(), kt, kh, 0, v.data_ptr(), vt, vh, 0, a.data_ptr(), b.data_ptr(),
               at if T > 1 else Hv, bt if T > 1 else Hv, 0 if A_log is None else A_log.data_ptr(),
               0 if dt_bias is None else dt_bias.data_ptr(), state.data_ptr(), 0 if slots is None else slots.data_ptr(),
               starts.data_ptr(), T, Hk, Hv, Dk, Dv, n, st if n > 1 else Hv * Dk * Dv, B, act_of(a), normalize,
               Dk ** -0.5 if scale is None else scale)
    return d, (T, Hk, Hv, Dk, Dv, B)


@functools.lru_cache(256)
def gated_delta_workspace_bytes(T, B, Hk, Hv, Dk, max_len):
    n = ctypes.c_size_t()
    check(lib().sx_gated_delta_workspace_bytes(T, B, Hk, Hv, Dk, max_len, ctypes.byref(n)))
    return n.value


def gated_delta_workspace(q, v, starts, max_len):
    """A workspace for gated_delta calls of these shapes (one per stream; nothing in it outlives a call); None where such
    calls need none."""
    n = gated_delta_workspace_bytes(q.shape[0], starts.numel() - 1, q.shape[1], v.shape[1], q.shape[2], max_len)
    return torch.empty((n + 7) // 8, dtype=torch.int64, device=q.device) if n else None


def gated_delta(q, k, v, a, b, state, starts, max_len, slots=None, A_log=None, dt_bias=None, normalize=True, scale=None, out=None,
                ws=None, err=None, stream=None):
    """The gated delta rule: for each token of a sequence and value head S <- e^g S, u = beta (v - S^T k), S <- S + k u^T, o = S^T q.
    q, k [T, Hk, Dk] and v [T, Hv, Dv] BF16 (any token and head strides; Hv a multiple of Hk), divided by their lengths first
    (normalize), q times scale (1 / sqrt(Dk) unless given). Gates a, b [T, Hv] in BF16 or FP32: with A_log and dt_bias (FP32 [Hv])
    g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b), else g = a and beta = b (g of -1e4 and less: a full reset). starts int32
    [B + 1], not falling: sequence b's tokens are rows starts[b] .. starts[b + 1] - 1, at most max_len; state FP32 [states, Hv, Dk, Dv],
    number slots[b] (int32 [B]; None: b) its own, updated in place (zeros: a new sequence). Up to 16 tokens a sequence go one by one, more in chunks. ws:
    gated_delta_workspace(), made for the call unless given. Returns (out [T, Hv, Dv] BF16, err)."""
    dev = q.get_device()
    _together(dev, (k, v, a, b, state, starts, slots, A_log, dt_bias, out, ws, err))
    d, (T, Hk, Hv, Dk, Dv, B) = _delta(q, k, v, a, b, state, starts, slots, A_log, dt_bias, normalize, scale)
    if out is None:
        out = _empty(q, (T, Hv, Dv), _BF16, stream)
        o = _ROWS(out.data_ptr(), Hv * Dv, Dv, 0)
    elif out.dim() != 3 or out.shape[0] != T:
        _refuse("out is", tuple(out.shape))
    else:
        o = _head_rows("out", out, Hv, Dv)
    if ws is None:
        n = 0 if max_len <= 16 else gated_delta_workspace_bytes(T, B, Hk, Hv, Dk, max_len)  # steps need none
        ws = _empty(q, ((n + 7) // 8,), torch.int64, stream) if n else None
    elif not ws.is_contiguous():
        _refuse("ws must be contiguous and has strides", ws.stride())
    _is_err(err)
    _run(dev, lib().sx_gated_delta, d, max_len, o, _a(ws), 0 if ws is None else ws.numel() * ws.element_size(), _a(err),
         stream=stream)
    return out, err


def gated_delta_verify(q, k, v, a, b, state, starts, mask, max_new, slots=None, A_log=None, dt_bias=None, normalize=True, scale=None,
                       out=None, u=None, decay=None, err=None, stream=None):
    """gated_delta of drafted tokens, whose states must wait for the accepted path: state is only read. A sequence's tokens, at
    most max_new (up to 64), are a tree; mask int64 [T, 1] as tree_mask makes it. Returns (out [T, Hv, Dv] BF16, u FP32 [T, Hv, Dv],
    decay FP32 [T, Hv], err); u and decay (and k) are what gated_delta_commit takes."""
    dev = q.get_device()
    _together(dev, (k, v, a, b, state, starts, mask, slots, A_log, dt_bias, out, u, decay, err))
    d, (T, Hk, Hv, Dk, Dv, B) = _delta(q, k, v, a, b, state, starts, slots, A_log, dt_bias, normalize, scale)
    if mask.dtype != torch.int64 or mask.dim() != 2 or mask.shape[0] != T or mask.shape[1] < 1:
        _refuse("mask must be int64 [T, 1] and is", mask.dtype, tuple(mask.shape))
    if out is None:
        out = _empty(q, (T, Hv, Dv), _BF16, stream)
        o = _ROWS(out.data_ptr(), Hv * Dv, Dv, 0)
    elif out.dim() != 3 or out.shape[0] != T:
        _refuse("out is", tuple(out.shape))
    else:
        o = _head_rows("out", out, Hv, Dv)
    if u is None:
        u = _empty(q, (T, Hv, Dv), torch.float32, stream)
    else:
        _is("u", u, torch.float32, (T, Hv, Dv))
    if decay is None:
        decay = _empty(q, (T, Hv), torch.float32, stream)
    else:
        _is("decay", decay, torch.float32, (T, Hv))
    _is_err(err)
    _run(dev, lib().sx_gated_delta_verify, d, max_new, mask.data_ptr(), mask.stride(0) if T > 1 else 1, o,
         u.data_ptr(), decay.data_ptr(), _a(err), stream=stream)
    return out, u, decay, err


def gated_delta_commit(k, u, decay, state, starts, count, path=None, max_count=None, slots=None, err=None, stream=None):
    """The accepted path of a gated_delta_verify into the states, in place: its first count[b] (int32 [B]) tokens, number path[b, i]
    of the sequence (int32 [B, at most]; None: i) the i-th of them. k [T, Hk, Dk], u and decay as the verify had and gave them; all
    layers in one launch with k [layers, T, Hk, Dk], u [layers, T, Hv, Dv], decay [layers, T, Hv], state [layers, states, Hv, Dk,
    Dv]. Without a path max_count bounds the counts. Returns err. A sequence that cannot be committed as asked keeps its states."""
    dev, ks, us, ss = k.get_device(), k.shape, u.shape, state.shape
    layered = len(ks) == 4
    _together(dev, (u, decay, state, starts, count, path, slots, err))
    if len(ks) not in (3, 4) or len(us) != len(ks) or len(ss) != 4 + layered or starts.dim() != 1:
        _refuse("k, u and state are", tuple(ks), tuple(us), tuple(ss), "and not of one number of layers")
    T, Hk, Dk = ks[-3:] if layered else ks
    Tu, Hv, Dv = us[-3:] if layered else us
    layers, B, st, kt = ks[0] if layered else 1, starts.shape[0] - 1, state.stride(), k.stride()
    if (k.dtype is not _BF16 or kt[-1] != 1 or Tu != T or u.dtype is not _F32 or not u.is_contiguous() or layered and (us[0] != layers or ss[0] != layers)):
        _refuse("k must be BF16 [tokens, heads, dim] with dense rows and u FP32, contiguous, of its layers and tokens:", k.dtype, tuple(ks), kt, u.dtype, tuple(us), u.stride())
    if decay.dtype is not _F32 or decay.shape != us[:-1] or not decay.is_contiguous():
        _is("decay", decay, _F32, us[:-1])
    if state.dtype is not _F32 or ss[-3] != Hv or ss[-2] != Dk or ss[-1] != Dv or st[-3] != Dk * Dv or st[-2] != Dv or st[-1] != 1:
        _refuse(f"state must be FP32 [{'layers, ' if layered else ''}states, {Hv}, {Dk}, {Dv}], each dense, and is", state.dtype, tuple(ss), st)
    if (B < 1 or starts.dtype is not _I32 or count.dtype is not _I32 or count.shape != (B,) or not (starts.is_contiguous() and count.is_contiguous()) or
            slots is not None and (slots.dtype is not _I32 or slots.shape != (B,) or not slots.is_contiguous())):
        _is("starts", starts, _I32, (B + 1,)), _is("count", count, _I32, (B,)), slots is not None and _is("slots", slots, _I32, (B,))
    ld = 0
    if path is not None:
        if path.dtype is not _I32 or path.dim() != 2 or path.shape[0] != B or path.stride(1) != 1:
            _refuse("path must be int32 [batch, most tokens kept] with dense rows")
        most = path.shape[1]
        max_count = most if max_count is None else max_count
        ld = path.stride(0) if B > 1 else most
        if max_count > most:
            _refuse("max_count =", max_count, "is over the path's", most)
    elif max_count is None:
        _refuse("max_count is needed without a path")
    _is_err(err)
    states, one = ss[-4], Hv * Dk * Dv
    _run(dev, lib().sx_gated_delta_commit, _ROWS(k.data_ptr(), kt[-3], kt[-2], kt[0] if layered else 0), u.data_ptr(),
         decay.data_ptr(), layers, T, Hk, Hv, Dk, Dv, state.data_ptr(), st[0] if layered else 0, st[-4] if states > 1 else one, states, _a(slots), starts.data_ptr(), B, count.data_ptr(), max_count, _a(path), ld,
         _a(err), stream=stream)
    return err


# ---------------- acceptance by the target's probabilities ----------------

@functools.lru_cache(256)
def mtp_accept_sampled_workspace_bytes(T, B, n_valid, n_draft):
    n = ctypes.c_size_t()
    check(lib().sx_mtp_accept_sampled_workspace_bytes(T, B, n_valid, n_draft, ctypes.byref(n)))
    return n.value


def mtp_accept_sampled(logits, drafts, starts, u, temperature, max_rows, draft_logits=None, n_valid=None, tokens=None, count=None,
                       status=None, ws=None, stream=None):
    """Acceptance of drafted tokens by rejection sampling. Sequence b's rows are starts[b] .. starts[b + 1] - 1 (int32 [B + 1], at
    most max_rows) of logits [T, >= n_valid] (FP32 or BF16, any row stride); drafts int32 [T]: the token proposed behind a row (a
    sequence's last row has none); draft_logits [T, n_draft] in the logits' type: what it was drawn from (None: it was certain). Draft
    d of row t stays if u[t, 0] q(d) < p(d), p and q the softmax over temperature[b] (FP32 [B]); the first that does not is replaced by a
    token from max(p - q, 0), and behind the last comes one from p, both by u[t, 1]. u FP64 [T, 2] in [0, 1). temperature 0: the
    largest logits. Returns (tokens int32 [B, max_rows]: what is committed, then -1; count int32 [B], as kv_append and
    gated_delta_commit take it; status int32 [B]: 0, 1 + the row that has no distribution or draft, -1 impossible starts)."""
    dev, act, shape, lt = logits.get_device(), act_of(logits), logits.shape, logits.stride()
    if len(shape) != 2 or lt[1] != 1 or starts.dim() != 1:
        _refuse("logits must be [T, vocabulary] with dense rows and are", tuple(shape), lt, "starts [B + 1]:", tuple(starts.shape))
    T, width = shape
    n_valid, n_draft, dld, B = width if n_valid is None else n_valid, 0, 0, starts.shape[0] - 1
    _together(dev, (drafts, starts, u, temperature, draft_logits, tokens, count, status, ws))
    if n_valid > width:
        _refuse("n_valid =", n_valid, "is over the logits'", width)
    if (drafts.dtype is not _I32 or drafts.shape != (T,) or starts.dtype is not _I32 or u.dtype is not torch.float64 or u.shape != (T, 2) or
            temperature.dtype is not _F32 or temperature.shape != (B,) or
            not (drafts.is_contiguous() and starts.is_contiguous() and u.is_contiguous() and temperature.is_contiguous())):
        _is("drafts", drafts, _I32, (T,)), _is("starts", starts, _I32, (B + 1,)), _is("u", u, torch.float64, (T, 2))
        _is("temperature", temperature, _F32, (B,))
    if draft_logits is not None:
        if draft_logits.dtype is not logits.dtype or draft_logits.dim() != 2 or draft_logits.shape[0] != T or draft_logits.stride(1) != 1:
            _refuse("draft_logits must be", logits.dtype, f"[{T}, vocabulary] with dense rows and are", draft_logits.dtype, tuple(draft_logits.shape))
        n_draft = draft_logits.shape[1]
        dld = draft_logits.stride(0) if T > 1 else n_draft
    if tokens is None:
        tokens = _empty(drafts, (B, max_rows), _I32, stream)
    else:
        _is("tokens", tokens, _I32, (B, max_rows))
    if count is None:
        count = _empty(drafts, (B,), _I32, stream)
    else:
        _is("count", count, _I32, (B,))
    if status is None:
        status = _empty(drafts, (B,), _I32, stream)
    else:
        _is("status", status, _I32, (B,))
    if ws is None:
        ws = _empty(drafts, ((mtp_accept_sampled_workspace_bytes(T, B, n_valid, n_draft) + 7) // 8,), torch.int64, stream)
    elif not ws.is_contiguous():
        _refuse("ws must be contiguous and has strides", ws.stride())
    _run(dev, lib().sx_mtp_accept_sampled, logits.data_ptr(), lt[0] if T > 1 else width, T, n_valid,
         _a(draft_logits), dld, n_draft, act, drafts.data_ptr(), starts.data_ptr(), B, max_rows, u.data_ptr(), temperature.data_ptr(),
         tokens.data_ptr(), count.data_ptr(), status.data_ptr(), ws.data_ptr(), ws.numel() * ws.element_size(), stream=stream)
    return tokens, count, status
