"""The verify path as the reference's runtime strings the operators together (runtime/qwen4exp.cpp:1130-1160 for the
MoE sublayer at T >= kGroupedMinTokens, 1191-1210 for the head, serve/engine.cpp:592-610 for the accept loop), on
preallocated device buffers so a forward allocates nothing.
"""
import torch

from . import MOE_F32, SxError
from . import kernels as kx


class MoeVerifyLayer:
    """One MoE FFN sublayer. Weights: Wr FP32 [E, d], gate_up q4 [E * 2I, d], down q4 [E * d, I] (experts stacked,
    runtime/qwen4exp.cpp:126-129). At verify width (the shapes kernels.verify_supported takes) three launches:
    router projection -> routing + gate_up + SwiGLU (the tails of its compute units' shares balanced through a sync
    buffer the layer owns) -> down + combine (the sequence qwen4exp.cpp:1139-1163 runs below kGroupedMinTokens). Otherwise (or fused=False): router projection -> moe_router + moe_group_routes -> grouped
    gate_up with the SwiGLU epilogue -> grouped down + combine. routing (optional): a dict of moe_router_scored's score,
    bias, groups, top_groups, group_best, renorm and factor; the layer then routes by those scores (grouped experts at
    every width) and not by moe_router. The layer has one set of buffers: forwards on different streams have to be ordered."""

    def __init__(self, Wr, gate_up, down, E, k, max_tokens, act_dtype=torch.bfloat16, fused=True, routing=None):
        self.Wr, self.gate_up, self.down, self.E, self.k = Wr, gate_up, down, E, k
        self.d = gate_up.K
        self.I = down.K
        assert gate_up.N == E * 2 * self.I and down.N == E * self.d
        dev = Wr.device
        M, A = max_tokens, k
        self.M = M
        self.logits = torch.empty((M, E), dtype=torch.float32, device=dev)
        self.ids = torch.empty((M, A), dtype=torch.int32, device=dev)
        self.coef = torch.empty((M, A), dtype=torch.float32, device=dev)
        self.router_err = torch.zeros(4, dtype=torch.int32, device=dev)
        self.expert_err = torch.zeros(4, dtype=torch.int32, device=dev)
        self.ws = torch.empty(kx.route_workspace_bytes(M, A, E) // 4, dtype=torch.int32, device=dev)
        self.h = torch.empty((M, A, self.I), dtype=act_dtype, device=dev)
        self.h_sums = torch.empty((M * A, (self.I + 15) // 16), dtype=torch.float32, device=dev)
        self.partial = torch.empty((M * A, self.d), dtype=torch.float32, device=dev)
        self.y = torch.empty((M, self.d), dtype=act_dtype, device=dev)
        self.routing = routing
        self.fused = fused and act_dtype == torch.bfloat16 and routing is None
        # the gate_up pool's sync buffers, one per stream: launches on one buffer must run in order, which only one
        # stream guarantees
        self._syncs = {}
        self.plan = kx.verify_plan(dev)  # the routing gate_up hands to down (written and read in stream order)
        self._dev = dev

    def _sync_for(self, stream):
        key = (stream or torch.cuda.current_stream(self._dev)).cuda_stream
        if key not in self._syncs:
            with torch.cuda.stream(stream):  # zeroed in the stream's own order (None: the current one)
                self._syncs[key] = kx.verify_layer_sync(self._dev)
        return self._syncs[key]

    def _fused(self, M):
        return self.fused and kx.verify_supported(M, self.k, self.E, self.k, self.E, self.gate_up, self.down)

    def forward(self, x, stream=None):
        if self.Wr.is_cuda and self._dev.index != torch.cuda.current_device():
            with torch.cuda.device(self._dev):
                return self.forward(x, stream)
        M = x.shape[0]
        assert M <= self.M
        ws = self.ws if M == self.M else self.ws[:kx.route_workspace_bytes(M, self.k, self.E) // 4]
        kx.linear_f32w(x, self.Wr, y=self.logits[:M], stream=stream)
        if self._fused(M):
            kx.verify_gate_up(x, self.logits[:M], self.gate_up, self.E, self.k, ids=self.ids[:M], coef=self.coef[:M],
                              h=self.h[:M], router_err=self.router_err, expert_err=self.expert_err,
                              h_sums=self.h_sums, sync=self._sync_for(stream), plan=self.plan, stream=stream)
            kx.verify_down(self.h[:M], self.down, self.ids[:M], self.coef[:M], self.E, y=self.y[:M],
                           expert_err=self.expert_err, h_sums=self.h_sums, plan=self.plan, stream=stream)
            return self.y[:M]
        if self.routing is not None:
            kx.moe_router_scored(self.logits[:M], self.E, self.k, ids=self.ids[:M], coef=self.coef[:M],
                                 err=self.router_err, stream=stream, **self.routing)
            kx.group_routes(self.ids[:M], self.E, ws=ws, err=self.expert_err, stream=stream)
        elif M * self.k <= 2048:  # top-k + grouping in one launch
            kx.router_group(self.logits[:M], self.E, self.k, ws=ws, ids=self.ids[:M], coef=self.coef[:M],
                            router_err=self.router_err, expert_err=self.expert_err, stream=stream)
        else:
            kx.moe_router(self.logits[:M], self.E, self.k, ids=self.ids[:M], coef=self.coef[:M],
                          err=self.router_err, stream=stream)
            kx.group_routes(self.ids[:M], self.E, ws=ws, err=self.expert_err, stream=stream)
        kx.gather_grouped(x, self.gate_up, self.E, ws, M, self.k, swiglu=True, y=self.h[:M], stream=stream)
        kx.combine_grouped(self.h[:M], self.down, self.E, self.ids[:M], self.coef[:M], ws,
                           partial=self.partial[:M * self.k], y=self.y[:M], math=MOE_F32, stream=stream)
        return self.y[:M]

    def weight_bytes_touched(self, M=None):
        """Algorithmic bytes of the last forward: the distinct experts' gate_up + down rows, the router weight and
        the activations in and out (synchronizes to read the ids)."""
        M = self.M if M is None else M
        U = int(torch.unique(self.ids[:M]).numel())
        per_expert = (self.gate_up.nbytes() + self.down.nbytes()) // self.E
        act = M * self.d * self.y.element_size()
        return U, U * per_expert + self.Wr.numel() * 4 + 2 * act


class VerifyAttention:
    """The attention half of a verify layer: x + residual, RMS norm and FP8 codes in one launch -> FP8 query, key and value
    projection -> attention of the drafted tokens over the layer's paged cache and each other -> output projection (a
    q4 / q8 weight). norm_w BF16 [d]; qkv an Fp8Weight [(Hq + 2 Hkv) D, d], heads in that order; out_w a QWeight
    [d, Hq D]. rotate (optional): called with the BF16 views q [T, Hq, D] and k [T, Hkv, D] after the projection, to turn
    them by their positions in place, forward's stream being the current one. The drafted tokens' keys and values stay in
    k_new and v_new, the last forward's, until the next forward on its stream: what kv_append takes once the accepted path is
    known. Buffers for max_tokens and a workspace are kept for every stream that forward is called on (a captured graph has
    those of the stream that it was captured on), so forwards on different streams do not meet; residual, q8, scale, heads,
    att and y are the last forward's."""

    def __init__(self, norm_w, qkv, out_w, Hq, Hkv, D, max_tokens, max_seqs, max_new, eps=1e-6, rotate=None):
        assert qkv.N == (Hq + 2 * Hkv) * D and out_w.K == Hq * D and out_w.N == qkv.K == norm_w.numel()
        self.norm_w, self.qkv, self.out_w, self.Hq, self.Hkv, self.D = norm_w, qkv, out_w, Hq, Hkv, D
        self.M, self.max_seqs, self.max_new, self.eps, self.rotate = max_tokens, max_seqs, max_new, eps, rotate
        self._dev = norm_w.device
        self.err = torch.zeros(4, dtype=torch.int32, device=self._dev)
        self.k_new = self.v_new = None
        first = self._make_buffers()
        self._buffers, self._ws = {}, {}
        if norm_w.is_cuda:  # they come from the current stream's pool
            self._buffers[torch.cuda.current_stream(self._dev).cuda_stream] = first
        vars(self).update(first)

    def _make_buffers(self):
        dev, d, M = self._dev, self.qkv.K, self.M
        return dict(residual=torch.empty((M, d), dtype=torch.bfloat16, device=dev),
                    q8=torch.empty((M, d), dtype=torch.float8_e4m3fn, device=dev),
                    scale=torch.empty((M, d // 128), dtype=torch.float32, device=dev),
                    heads=torch.empty((M, self.Hq + 2 * self.Hkv, self.D), dtype=torch.bfloat16, device=dev),
                    att=torch.empty((M, self.Hq, self.D), dtype=torch.bfloat16, device=dev),
                    y=torch.empty((M, d), dtype=torch.bfloat16, device=dev))

    def _ws_for(self, stream):
        """The stream's workspace. The stream's buffers become the layer's."""
        key = (stream or torch.cuda.current_stream(self._dev)).cuda_stream
        if key not in self._ws:
            with torch.cuda.device(self._dev), torch.cuda.stream(stream):  # from the stream's pool (None: the current one's)
                n = kx.tree_attention_workspace_bytes(self.max_seqs, self.Hq, self.Hkv, self.D, self.max_new)
                self._ws[key] = torch.empty((n + 7) // 8, dtype=torch.int64, device=self._dev)
                if key not in self._buffers:
                    self._buffers[key] = self._make_buffers()
        vars(self).update(self._buffers[key])
        return self._ws[key]

    def forward(self, x, residual, k_cache, v_cache, table, lens, starts, mask, k_scale=1.0, v_scale=1.0, stream=None):
        """x, residual (None in the first layer) BF16 [T, d]; the rest as tree_attention takes them. Returns (y [T, d],
        the sum x + residual). Runs on the layer's device, whichever is current."""
        if self.norm_w.is_cuda and self._dev.index != torch.cuda.current_device():
            with torch.cuda.device(self._dev):
                return self.forward(x, residual, k_cache, v_cache, table, lens, starts, mask, k_scale, v_scale, stream)
        T = x.shape[0]
        assert T <= self.M and lens.numel() <= self.max_seqs
        ws = self._ws_for(stream)
        res = None if residual is None else self.residual[:T]
        kx.add_rms_norm_fp8(x, self.norm_w, self.eps, residual=residual, residual_out=res, q=self.q8[:T],
                            scale=self.scale[:T], stream=stream)
        heads = self.heads[:T]
        kx.linear_fp8(self.q8[:T], self.scale[:T], self.qkv, y=heads.view(T, -1), stream=stream)
        q, self.k_new, self.v_new = heads.split([self.Hq, self.Hkv, self.Hkv], dim=1)
        if self.rotate is not None:
            with torch.cuda.stream(stream):  # the projection and the attention run there (None: the current one)
                self.rotate(q, self.k_new)
        kx.tree_attention(q, self.k_new, self.v_new, k_cache, v_cache, table, lens, starts, mask, self.max_new,
                          k_scale=k_scale, v_scale=v_scale, out=self.att[:T], ws=ws, err=self.err,
                          stream=stream)
        kx.linear(self.att[:T].view(T, -1), self.out_w, y=self.y[:T], stream=stream)
        return self.y[:T], x if residual is None else res


class VerifyTail:
    """The verify head: q8 LM head [V, d] -> FP32 logits [M, V] -> logits_topk (k candidates) -> device acceptance."""

    def __init__(self, lm_head, n_valid, k_cands, max_rows):
        self.w, self.n_valid, self.kc = lm_head, n_valid, k_cands
        dev = lm_head.q.device
        self.logits = torch.empty((max_rows, lm_head.N), dtype=torch.float32, device=dev)
        self.cands = torch.empty((max_rows, k_cands, 2), dtype=torch.int32, device=dev)
        self.nan = torch.empty(max_rows, dtype=torch.int32, device=dev)
        self.ws = torch.empty(kx.topk_workspace_bytes(max_rows, n_valid, k_cands) // 8 + 1, dtype=torch.int64,
                              device=dev)
        self.out = torch.empty(2 + max_rows, dtype=torch.int32, device=dev)
        # top-k and acceptance as one launch where the first level's candidates fit one block a row
        try:
            self.tail_ws = kx.verify_tail_workspace(max_rows, n_valid, k_cands, dev)
        except SxError:  # more first-level candidates a row than one block reduces: two launches
            self.tail_ws = None

    def forward(self, h, drafts, u, temperature, top_k, top_p, stream=None):
        M = h.shape[0]
        kx.linear(h, self.w, out_act=0, y=self.logits[:M], stream=stream)
        out = self.out[:2 + drafts.numel() + 1]
        if self.tail_ws is not None and M >= drafts.numel() + 1:
            kx.verify_tail(self.logits[:M], self.n_valid, self.kc, self.tail_ws, drafts=drafts, u=u,
                           temperature=temperature, top_k=top_k, top_p=top_p, cands=self.cands[:M],
                           nan=self.nan[:M], out=out, stream=stream)
            return out
        kx.logits_topk(self.logits[:M], self.n_valid, self.kc, ws=self.ws, out=self.cands[:M], nan=self.nan[:M],
                       stream=stream)
        return kx.mtp_accept(self.cands[:M], self.nan[:M], drafts, u, temperature, top_k, top_p, self.n_valid,
                             out=out, stream=stream)
