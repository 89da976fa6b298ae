"""Batched frozen-state decoding over ring-buffer SWA caches.

The reference decodes one request at a time, either eagerly (``uTTTModel.stream_generate``,
``model/uttt_model.py:966-1179``) or through ``CUDAGraphDecoder`` (``engine/inference.py:71-302``),
whose captured step writes the new key/value into ring slot ``pos mod window``, masks the slots
that are not yet valid and reads each layer's fast weights through activation-dtype copies.

``BatchedDecoder`` runs N independent requests in one step: every request keeps its own fp32
fast-weight master state (read through per-request activation-dtype copies), its own position
and its own ring slots.  One step is, per layer: RMSNorm -> packed QKV GEMM -> ``uttt_swa_decode``
(RoPE at each request's position, ring write, window attention) -> output GEMM -> RMSNorm ->
query projection -> per-request fast-weight readout (``uttt_swiglu_readout`` over the stacked
copies) -> output GEMM; then the final norm, the LM head and the next token's selection, greedy or
sampled (``set_sampling``), all on the device, so ``capture()`` can record the whole step into one
HIP graph.

Beside the step (not in the reference's decoders): ``verify`` runs a tree of drafted tokens per
request through the model at once, without writing the rings, ``commit`` makes a path of it part
of the requests, ``speculate_greedy`` does both, and ``fork`` lets requests take over others'
caches.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch
import torch.nn.functional as F

from . import kernels as K
from .layer import FastWeightState, linear_residual
from .model import BOS_ID, PAD_ID, UNK_ID, uTTTModel

Tensor = torch.Tensor


class BatchedDecoder:
    """N requests, one token each per step, frozen fast weights (decode never writes them)."""

    def __init__(self, model: uTTTModel, states: Sequence[FastWeightState], max_positions: int = 8192):
        if model.training:
            raise ValueError("call model.eval() before decoding")
        if not states:
            raise ValueError("need at least one request state")
        self.model = model
        self.n = len(states)
        dev = model.tok_embeddings.weight.device
        if dev.type != "cuda":
            raise ValueError("BatchedDecoder needs the model on the GPU")
        self.device = dev
        self.dtype = model.tok_embeddings.weight.dtype
        for st in states:
            if st.w_up.shape[0] != 1:
                raise ValueError("each request state must hold one row (batch 1)")
        ln_w, ln_b = states[0].ln_weight, states[0].ln_bias
        for st in states[1:]:
            if not (torch.equal(st.ln_weight, ln_w) and torch.equal(st.ln_bias, ln_b)):
                raise ValueError("batched decoding needs one shared LayerNorm pair for all requests")
        self.ln_weight = ln_w.detach().float().contiguous()
        self.ln_bias = ln_b.detach().float().contiguous()
        # per-request read copies in the activation dtype (reference inference_read_weights,
        # model/uttt_layer.py:648-668): same operands the reference's bf16 matmuls see
        with torch.no_grad():
            self.w_up = torch.cat([st.w_up.detach() for st in states]).to(self.dtype).contiguous()
            self.w_gate = torch.cat([st.w_gate.detach() for st in states]).to(self.dtype).contiguous()
            self.w_down = torch.cat([st.w_down.detach() for st in states]).to(self.dtype).contiguous()
        attn = model.layers[0].attn
        self.window, self.hkv, self.hd, self.heads = attn.window_size, attn.n_kv_heads, attn.head_dim, attn.n_heads
        self.sinks = attn.sinks
        # every layer's slots in one tensor: commits and forks take all layers in one launch
        self.slots = self.sinks + self.window
        self.k_rings, self.v_rings = (torch.zeros((len(model.layers), self.n, self.hkv, self.slots, self.hd),
                                                  dtype=self.dtype, device=dev) for _ in range(2))
        self.rings = [(self.k_rings[li], self.v_rings[li]) for li in range(len(model.layers))]
        self.cos, self.sin = attn.rope.tables(max_positions, dev)
        self.positions = torch.zeros(self.n, dtype=torch.int64, device=dev)
        self.host_positions = [0] * self.n
        self.tokens = torch.zeros(self.n, dtype=torch.int64, device=dev)
        self.logits: Optional[Tensor] = None
        self.next_tokens: Optional[Tensor] = None
        self.logprobs: Optional[Tensor] = None  # of the sampled next tokens, after ``set_sampling``
        self._sampling: Optional[dict] = None
        self._nodes: Optional[Tuple[Tensor, Tensor]] = None  # the last verified trees' keys / values
        self._graph = None
        self._graph_logits: Optional[Tensor] = None  # where the recorded step leaves its logits
        self._ws_attn = torch.zeros(1, dtype=torch.uint8, device=dev)
        self._ws_read = torch.zeros(1, dtype=torch.uint8, device=dev)
        self._states = list(states)
        self._key = self._state_key(states)
        self._folds = {}
        d_model = model.config.d_model
        self._fused_readout = self.dtype == torch.bfloat16 and d_model <= 2048 and all(
            (blk.uttt.q_norm.eps or 0.0) > 0.0 for blk in model.layers)
        self._counters = torch.zeros(self.n, dtype=torch.int32, device=dev)  # left zero by every readout

    # ------------------------------------------------------------------ prefill
    @torch.no_grad()
    def prefill(self, prompts: Sequence[Tensor]) -> Tensor:
        """Frozen prefill of each request's prompt (its own state), then load the last
        ``window`` keys/values into the ring slots.  Returns the next-token logits (N, V)."""
        if len(prompts) != self.n:
            raise ValueError(f"expected {self.n} prompts, got {len(prompts)}")
        self._nodes = None
        out_logits = []
        for i, (ids, st) in enumerate(zip(prompts, self._states)):
            ids = ids.to(self.device).view(1, -1)
            if ids.shape[1] == 0:
                raise ValueError("prompts must be non-empty")
            out = self.model(ids, fast_state=st, update_fast_weights=False, logits_to_keep=1)
            self._load_request(i, out.kv_caches, ids.shape[1])
            out_logits.append(out.logits[:, -1, :])
        self.positions.copy_(torch.tensor(self.host_positions, dtype=torch.int64))
        return torch.cat(out_logits, dim=0)

    def _cached_slots(self, cached: int, length: int) -> Tensor:
        """The slots of the ``cached`` rows of a request of ``length`` tokens: its first tokens, as
        far as they are sinks, then its last ones.  Token p has slot p while p < sinks and
        sinks + (p - sinks) mod window from there."""
        first = min(self.sinks, cached)
        tokens = torch.arange(length - (cached - first), length, device=self.device)
        recent = torch.where(tokens < self.sinks, tokens, self.sinks + (tokens - self.sinks) % self.window)
        return torch.cat((torch.arange(first, device=self.device), recent)) if first else recent

    def _load_request(self, i: int, kv_caches, length: int) -> None:
        """Request i's ring slots from a frozen prefill's per-layer caches (the last <= window
        rotated keys / values of ``length`` tokens, behind the sinks)."""
        if len(kv_caches) != len(self.rings):
            raise ValueError(f"expected {len(self.rings)} layer caches, got {len(kv_caches)}")
        for (kr, vr), (k, v) in zip(self.rings, kv_caches):
            cached = k.shape[2]
            if (k.shape != (1, self.hkv, cached, self.hd) or v.shape != k.shape or cached > min(length, self.slots)
                    or cached < min(length, self.slots - 1)):
                raise ValueError("a cache must be (1, n_kv_heads, min(length, sinks + window) or sinks + window - 1, "
                                 "head_dim)")
            slots = self._cached_slots(cached, length)
            kr[i].index_copy_(1, slots, k[0].to(device=self.device, dtype=kr.dtype))
            vr[i].index_copy_(1, slots, v[0].to(device=self.device, dtype=vr.dtype))
        self.host_positions[i] = int(length)

    @torch.no_grad()
    def reset(self, kv_caches_per_request: Sequence, lengths: Sequence[int]) -> None:
        """Start again from other prompts' frozen-prefill caches (same requests and states):
        the rings, positions and buffers keep their addresses, so a captured step stays valid."""
        if len(kv_caches_per_request) != self.n or len(lengths) != self.n:
            raise ValueError(f"expected caches and lengths for {self.n} requests")
        self._nodes = None
        for kr, vr in self.rings:
            kr.zero_()
            vr.zero_()
        for i, (caches, length) in enumerate(zip(kv_caches_per_request, lengths)):
            if length < 1:
                raise ValueError("a request needs at least one prompt token")
            self._load_request(i, caches, int(length))
        self.positions.copy_(torch.tensor(self.host_positions, dtype=torch.int64))

    @torch.no_grad()
    def export_kv_caches(self, i: int = 0) -> List:
        """Request i's per-layer caches in the eager layout (the sinks, then the last rotated keys /
        values up to the window in token order), e.g. to continue a decode eagerly."""
        pos = self.host_positions[i]
        slots = self._cached_slots(min(pos, self.slots), pos)
        return [(kr[i:i + 1].index_select(2, slots), vr[i:i + 1].index_select(2, slots)) for kr, vr in self.rings]

    def matches(self, model: uTTTModel, states: Sequence[FastWeightState]) -> bool:
        """Whether this decoder's read copies and LayerNorm pair still stand for ``states`` of
        ``model`` (same tensors, unchanged versions), so it can be ``reset`` and reused."""
        return model is self.model and len(states) == self.n and self._state_key(states) == self._key

    @staticmethod
    def _state_key(states: Sequence[FastWeightState]) -> tuple:
        return tuple((t.data_ptr(), t._version, t.dtype) for st in states
                     for t in (st.w_up, st.w_gate, st.w_down, st.ln_weight, st.ln_bias))

    # ------------------------------------------------------------------ one step
    def _folded(self, weight: Tensor, norm) -> Tensor:
        """W diag(g) for an RMSNorm ``norm`` applied to W's input (formed in fp32, rounded
        once), rebuilt when either changes."""
        key = (weight.data_ptr(), weight._version, norm.weight.data_ptr(), norm.weight._version)
        hit = self._folds.get(id(weight))
        if hit is None or hit[0] != key:
            fold = (weight.detach().float() * norm.weight.detach().float()[None, :]).to(weight.dtype).contiguous()
            hit = (key, fold)
            self._folds[id(weight)] = hit
        return hit[1]

    def _linear(self, x: Tensor, weight: Tensor, residual: Optional[Tensor] = None, norm=None) -> Tensor:
        """norm(x) W^T (+ residual, updated in place): ``uttt_skinny_linear`` for bf16 steps of
        at most 64 requests (the RMSNorm folded in), the norm and the library GEMM otherwise."""
        skinny = (x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and x.shape[0] <= 64
                  and weight.shape[0] % 32 == 0 and x.shape[1] % 64 == 0 and x.stride(1) == 1
                  and weight.is_contiguous() and (norm is None or (norm.eps or 0.0) > 0.0))
        if skinny:
            if norm is None:
                return K.skinny_linear(x, weight, out=residual, residual=residual)
            return K.skinny_linear(x, self._folded(weight, norm), out=residual, residual=residual,
                                   x_eps=norm.eps)
        if norm is not None:
            x = norm(x)
        if residual is not None:
            return linear_residual(residual, x, weight)
        return F.linear(x, weight)

    def _step_body(self) -> None:
        m = self.model
        n = self.n
        h = F.embedding(self.tokens, m.tok_embeddings.weight)  # (N, D)
        for li, block in enumerate(m.layers):
            attn = block.attn
            qkv = self._linear(h, attn.packed_qkv().to(h.dtype), norm=block.attn_norm)  # (N, (H + 2 Hkv) hd)
            hq = self.heads * self.hd
            hk = self.hkv * self.hd
            q = qkv[:, :hq].view(n, self.heads, self.hd)
            k = qkv[:, hq:hq + hk].view(n, self.hkv, self.hd)
            v = qkv[:, hq + hk:].view(n, self.hkv, self.hd)
            kr, vr = self.rings[li]
            att = K.swa_decode(q, k, v, kr, vr, self.positions, self.cos, self.sin, workspace=self._ws_attn,
                               sinks=self.sinks)
            h = self._linear(att.reshape(n, -1), attn.wo.weight, residual=h)
            y = self._linear(h, block.uttt.w_q.weight, norm=block.uttt_norm)
            qn = block.uttt.q_norm
            # every layer reads the same per-request copies: odd layers walk them backwards, so
            # each readout starts on the lines the previous one left in the infinity cache
            rev = li % 2 == 1
            if self._fused_readout:  # q_norm, readout, LayerNorm and residual in one launch
                r = K.swiglu_readout(y.view(n, 1, -1), self.w_up, self.w_gate, self.w_down, self.ln_weight,
                                     self.ln_bias, m.fast_weight_pool.eps, workspace=self._ws_read,
                                     x_norm=(qn.weight, qn.eps), row_counters=self._counters, sweep_reverse=rev)
            else:
                uq = F.rms_norm(y, (h.shape[-1],), qn.weight.to(h.dtype), qn.eps)
                r = K.swiglu_readout(uq.view(n, 1, -1), self.w_up, self.w_gate, self.w_down, self.ln_weight,
                                     self.ln_bias, m.fast_weight_pool.eps, workspace=self._ws_read,
                                     sweep_reverse=rev)
            h = self._linear(r.view(n, -1), block.uttt.w_o.weight, residual=h)
        logits = self._linear(h, m.lm_head.weight, norm=m.norm)
        self.logits = logits
        # temperature-0 selection: PAD / BOS / UNK and ids past the active vocabulary excluded,
        # written straight into the next step's input (stepping with `next_tokens` copies
        # nothing), and the positions advance in the same launch
        if self._sampling is None:
            self.next_tokens = K.greedy_select(logits, (PAD_ID, BOS_ID, UNK_ID), self._active_limit(logits),
                                               out=self.tokens, advance=self.positions)
        else:
            self._sample(logits, advance=self.positions)

    def _active_limit(self, logits: Tensor) -> Optional[int]:
        limit = self.model.active_vocab_limit
        return limit if limit < logits.shape[-1] else None

    def _sample(self, logits: Tensor, advance: Optional[Tensor] = None) -> None:
        s = self._sampling
        self.next_tokens, _ = K.sample_select(logits, s["uniforms"], s["temperature"], s["top_k"], s["top_p"],
                                              s["min_p"], (PAD_ID, BOS_ID, UNK_ID), self._active_limit(logits),
                                              out=self.tokens, logprobs=self.logprobs, advance=advance)

    def _warm_workspaces(self) -> None:
        from . import _native as N
        lib = N.load_library()
        if self.sinks:
            code = N.DTYPE_BF16 if self.dtype == torch.bfloat16 else N.DTYPE_F32
            nbytes = lib.uttt_swa_tree_workspace(self.n, self.heads, self.hkv, 1, self.hd, self.slots, code)
        else:
            nbytes = lib.uttt_swa_decode_workspace(self.n, self.heads, self.hkv, self.hd, self.window)
        self._ws_attn = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=self.device)
        d = self.model.config.d_model
        ff = self.model.config.d_ff_fast
        code = N.DTYPE_BF16 if self.dtype == torch.bfloat16 else N.DTYPE_F32
        self._ws_read = torch.zeros(max(N.load_library().uttt_readout_workspace(self.n, 1, d, ff, code), 1),
                                    dtype=torch.uint8, device=self.device)

    @torch.no_grad()
    def capture(self) -> None:
        """Record one step into a HIP graph (after ``prefill``, or between steps); ``step`` then replays it.  What the
        decoder holds stays as it was: caches, positions, the tokens chosen last and their logits."""
        self._warm_workspaces()
        held = [t for t in (self.positions, self.tokens, self.logprobs, self.k_rings, self.v_rings) if t is not None]
        saved = [t.clone() for t in held]
        chosen, logits = self.next_tokens, self.logits
        self._step_body()  # warm-up outside the graph (packs, tables, allocator)
        torch.cuda.synchronize()
        for t, t0 in zip(held, saved):
            t.copy_(t0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step_body()
        torch.cuda.synchronize()
        # capture ran no kernels: the logits recorded last are none yet
        self._graph, self._graph_logits = graph, self.logits
        self.next_tokens, self.logits = chosen, logits

    @torch.no_grad()
    def step(self, tokens: Tensor) -> Tensor:
        """Append one token per request; returns the logits (N, V) for the next position."""
        if tokens.shape != (self.n,):
            raise ValueError(f"tokens must be ({self.n},)")
        limit = self.cos.shape[0]
        if max(self.host_positions) >= limit:
            raise ValueError("a request reached the end of the RoPE table")
        if tokens.data_ptr() != self.tokens.data_ptr():
            self.tokens.copy_(tokens)
        self._nodes = None
        if self._sampling is not None:  # ahead of the step, so that a replay draws new ones
            self._sampling["uniforms"].uniform_(generator=self._sampling["generator"])
        if self._graph is not None:
            self._graph.replay()
            self.next_tokens, self.logits = self.tokens, self._graph_logits
        else:
            if self._ws_attn.numel() == 1:
                self._warm_workspaces()
            self._step_body()
        self.host_positions = [p + 1 for p in self.host_positions]
        return self.logits

    @torch.no_grad()
    def generate_greedy(self, first_logits: Tensor, steps: int) -> Tensor:
        """Greedy tokens (N, steps) continuing from ``first_logits`` (no EOS stop)."""
        if self._sampling is not None:
            raise ValueError("the decoder samples; set_sampling(None) makes its choices greedy again")
        m = self.model
        work = first_logits.float().clone()
        work[:, [PAD_ID, BOS_ID, UNK_ID]] = float("-inf")
        if m.active_vocab_limit < work.shape[-1]:
            work[:, m.active_vocab_limit:] = float("-inf")
        tok = work.argmax(dim=-1)
        out = [tok]
        for _ in range(steps - 1):
            self.step(tok)
            tok = self.next_tokens  # already the next step's input
            out.append(tok.clone())
        return torch.stack(out, dim=1)

    # ------------------------------------------------------------------ sampling
    @torch.no_grad()
    def set_sampling(self, temperature: Union[None, float, Sequence[float]], top_k: Union[int, Sequence[int]] = 0,
                     top_p: Union[float, Sequence[float]] = 1.0, min_p: Union[float, Sequence[float]] = 0.0,
                     generator: Optional[torch.Generator] = None) -> None:
        """Let every step choose its next tokens by sampling (``kernels.sample_select``), each setting
        one number or one per request; ``temperature`` None goes back to greedy choices.  The
        uniforms come from ``generator`` (of the model's device; the default one otherwise), drawn ahead of each
        step, so that a captured step draws new ones on each replay.  Settings changed later
        reach a captured step; changing between greedy and sampled drops it (``capture`` again)."""
        if temperature is None:
            if self._sampling is not None:
                self._sampling, self.logprobs, self._graph = None, None, None
            return
        rows = {}
        for name, value, low, high in (("temperature", temperature, 0.0, float("inf")), ("top_k", top_k, 0, 2 ** 31 - 1),
                                       ("top_p", top_p, 0.0, 1.0), ("min_p", min_p, 0.0, 1.0)):
            values = [value] * self.n if isinstance(value, (int, float)) else list(value)
            if len(values) != self.n:
                raise ValueError(f"{name} must be one number or one per request")
            if not all(low <= v <= high and v != float("inf") for v in values):
                raise ValueError(f"{name} must be finite, at least {low} and at most {high}")
            if name == "top_p" and min(values) <= 0.0:
                raise ValueError("top_p must be above 0")
            rows[name] = torch.tensor(values, dtype=torch.int32 if name == "top_k" else torch.float32)
        if self._sampling is None:
            self._sampling = {name: t.to(self.device) for name, t in rows.items()}
            self._sampling["uniforms"] = torch.zeros(self.n, dtype=torch.float32, device=self.device)
            self.logprobs = torch.zeros(self.n, dtype=torch.float32, device=self.device)
            self._graph = None
        else:
            for name, t in rows.items():
                self._sampling[name].copy_(t)
        self._sampling["generator"] = generator

    @torch.no_grad()
    def generate_sampled(self, first_logits: Tensor, steps: int) -> Tuple[Tensor, Tensor]:
        """Sampled tokens (N, steps) continuing from ``first_logits``, and the logarithms (N, steps) of
        the probabilities they were chosen with (no EOS stop; after ``set_sampling``)."""
        if self._sampling is None:
            raise ValueError("set_sampling comes first")
        self._sampling["uniforms"].uniform_(generator=self._sampling["generator"])
        self._sample(first_logits)
        out, logprobs = [self.tokens.clone()], [self.logprobs.clone()]
        for _ in range(steps - 1):
            self.step(self.tokens)
            out.append(self.tokens.clone())
            logprobs.append(self.logprobs.clone())
        return torch.stack(out, dim=1), torch.stack(logprobs, dim=1)

    # ------------------------------------------------------------------ drafted tokens
    @torch.no_grad()
    def verify(self, tokens: Tensor, parents: Optional[Tensor] = None, counts: Optional[Tensor] = None) -> Tensor:
        """The logits (N, T, V) behind every node of a tree of drafted tokens per request, all nodes
        at once: ``tokens`` (N, T) int64, T <= 64, ``parents`` (N, T) int32 (-1: the node follows the request's
        tokens so far, else an earlier node; None: each follows the one before it), ``counts`` (N,) int32 nodes that
        exist per request (None: T; the logits behind them mean nothing, and their tokens must be ids of
        the vocabulary all the same).  Neither the rings nor the positions change: ``commit`` makes a
        path of the tree part of each request."""
        if tokens.dim() != 2 or tokens.shape[0] != self.n or not 1 <= tokens.shape[1] <= K.N.MAX_TREE_NODES:
            raise ValueError(f"tokens must be ({self.n}, 1 to {K.N.MAX_TREE_NODES})")
        nodes = tokens.shape[1]
        if max(self.host_positions) + nodes > self.cos.shape[0]:
            raise ValueError("a request's drafted tokens reach past the end of the RoPE table")
        m, n = self.model, self.n
        parents = None if parents is None else parents.to(device=self.device, dtype=torch.int32).contiguous()
        counts = None if counts is None else counts.to(device=self.device, dtype=torch.int32).contiguous()
        shape = (len(m.layers), n, nodes, self.hkv, self.hd)
        k_nodes, v_nodes = (torch.empty(shape, dtype=self.dtype, device=self.device) for _ in range(2))
        if parents is not None or counts is not None:  # nodes that are not computed: loud, should they be committed
            k_nodes.fill_(float("nan"))
            v_nodes.fill_(float("nan"))
        h = F.embedding(tokens.to(self.device).reshape(-1), m.tok_embeddings.weight)  # (N T, D)
        hq, hk = self.heads * self.hd, self.hkv * self.hd
        read_ws = None
        for li, block in enumerate(m.layers):
            attn = block.attn
            qkv = self._linear(h, attn.packed_qkv().to(h.dtype), norm=block.attn_norm).view(n, nodes, -1)
            q = qkv[..., :hq].unflatten(-1, (self.heads, self.hd))
            k = qkv[..., hq:hq + hk].unflatten(-1, (self.hkv, self.hd))
            v = qkv[..., hq + hk:].unflatten(-1, (self.hkv, self.hd))
            att, _, _ = K.swa_tree(q, k, v, *self.rings[li], self.positions, parents, self.cos, self.sin, self.sinks,
                                   counts, node_outputs=(k_nodes[li], v_nodes[li]))
            h = self._linear(att.view(n * nodes, -1), attn.wo.weight, residual=h)
            y = self._linear(h, block.uttt.w_q.weight, norm=block.uttt_norm)
            qn = block.uttt.q_norm
            uq = F.rms_norm(y, (h.shape[-1],), qn.weight.to(h.dtype), qn.eps).view(n, nodes, -1)
            if read_ws is None:
                read_ws = K.readout_workspace(uq, self.w_up)
            r = K.swiglu_readout(uq, self.w_up, self.w_gate, self.w_down, self.ln_weight, self.ln_bias,
                                 m.fast_weight_pool.eps, workspace=read_ws, sweep_reverse=li % 2 == 1)
            h = self._linear(r.view(n * nodes, -1), block.uttt.w_o.weight, residual=h)
        logits = self._linear(h, m.lm_head.weight, norm=m.norm)
        self._nodes = (k_nodes, v_nodes)
        return logits.view(n, nodes, -1)

    @torch.no_grad()
    def commit(self, nodes: Tensor, counts: Tensor) -> None:
        """Append a path of the last verified trees to each request: the tokens of its nodes
        nodes[n, :counts[n]], from the first behind the request's tokens on, each the parent of the next (``nodes``
        (N, A) and ``counts`` (N,), on any device; the counts are read back).  A tree is committed once.  The next token is
        the caller's to choose, from ``verify``'s logits: ``self.tokens`` and ``self.logits`` stay the last step's."""
        if self._nodes is None:
            raise ValueError("commit follows verify, once, before anything else changes the requests")
        k_nodes, v_nodes = self._nodes
        if nodes.dim() != 2 or nodes.shape[0] != self.n or counts.shape != (self.n,):
            raise ValueError(f"nodes must be ({self.n}, A) and counts ({self.n},)")
        path, taken = nodes.to("cpu", torch.int64), counts.to("cpu", torch.int64).tolist()
        if min(taken) < 0 or max(taken) > path.shape[1]:
            raise ValueError("counts must be at least 0 and at most the columns of nodes")
        used = path[torch.arange(path.shape[1])[None, :] < torch.tensor(taken)[:, None]]
        if used.numel() and not 0 <= int(used.min()) <= int(used.max()) < k_nodes.shape[2]:
            raise ValueError("nodes must be nodes of the verified trees")
        self._nodes = None
        K.kv_commit(k_nodes, v_nodes, path.to(device=self.device, dtype=torch.int32),
                    torch.tensor(taken, dtype=torch.int32).to(self.device), self.k_rings, self.v_rings, self.positions,
                    self.sinks, advance=True)
        self.host_positions = [p + t for p, t in zip(self.host_positions, taken)]

    @torch.no_grad()
    def speculate_greedy(self, tokens: Tensor, parents: Optional[Tensor] = None,
                         counts: Optional[Tensor] = None) -> List[List[int]]:
        """One round of greedy decoding with drafted tokens: node 0 of each request's tree is its next token,
        chosen already, the others descend from it.  Verifies the trees, takes in each the longest path from
        node 0 whose every token is the greedy choice behind its parent, commits it and returns, per request, the
        drafted tokens taken and the greedy choice behind the last of them (the next round's node 0, in
        ``self.tokens`` too, with ``self.logits`` what it was chosen from): the tokens that single steps would give,
        as far as the products of more rows at once, and in bf16 the tree's rotations (rounded once, a step's without
        sinks after each operation), round alike.  Trees and the choices behind them are read back.  Refused, as
        ``generate_greedy`` is, while the decoder samples."""
        if self._sampling is not None:
            raise ValueError("the decoder samples; set_sampling(None) makes its choices greedy again")
        if tokens.dim() != 2 or tokens.shape[0] != self.n or tokens.shape[1] < 1:
            raise ValueError(f"tokens must be ({self.n}, nodes)")
        up = (torch.arange(-1, tokens.shape[1] - 1).expand(self.n, -1) if parents is None else parents.cpu()).tolist()
        held = [tokens.shape[1]] * self.n if counts is None else counts.tolist()
        if min(held) < 1 or max(held) > tokens.shape[1] or any(
                row[0] != -1 or any(not 0 <= p < t for t, p in enumerate(row[1:c], 1)) for row, c in zip(up, held)):
            raise ValueError("node 0 is each tree's root, and every other node's parent is an earlier node")
        logits = self.verify(tokens, parents, counts)
        n, nodes, vocab = logits.shape
        choice = K.greedy_select(logits.view(n * nodes, vocab), (PAD_ID, BOS_ID, UNK_ID),
                                 self._active_limit(logits)).view(n, nodes).tolist()
        drafted = tokens.tolist()
        paths = []
        for i in range(n):
            depth, deepest = [1] + [0] * (nodes - 1), 0  # of the nodes that agree with the choices; 0: not one
            for t in range(1, held[i]):
                if depth[up[i][t]] and drafted[i][t] == choice[i][up[i][t]]:
                    depth[t] = depth[up[i][t]] + 1
                    deepest = t if depth[t] > depth[deepest] else deepest
            path = [deepest]
            while path[-1] > 0:
                path.append(up[i][path[-1]])
            paths.append(path[::-1])
        longest = max(len(p) for p in paths)
        self.commit(torch.tensor([p + [0] * (longest - len(p)) for p in paths]), torch.tensor([len(p) for p in paths]))
        self.tokens.copy_(torch.tensor([choice[i][p[-1]] for i, p in enumerate(paths)]))
        last = torch.tensor([i * nodes + p[-1] for i, p in enumerate(paths)])
        self.next_tokens, self.logits = self.tokens, logits.view(n * nodes, vocab).index_select(0, last.to(self.device))
        return [[drafted[i][t] for t in p[1:]] + [choice[i][p[-1]]] for i, p in enumerate(paths)]

    # ------------------------------------------------------------------ requests taken over
    @torch.no_grad()
    def fork(self, sources: Sequence[int]) -> None:
        """Request i goes on from request sources[i], as that was before the call: its cache and
        position (``kernels.kv_fork``, in place), the token chosen last with its log-probability, its logits
        and its fast weights.  Sampling settings stay with the slot.  Buffers keep their addresses, so a
        captured step stays valid."""
        src = [int(s) for s in sources]
        if len(src) != self.n or min(src) < 0 or max(src) >= self.n:
            raise ValueError(f"sources must be {self.n} requests' indexes")
        self._nodes = None
        index = torch.tensor(src, dtype=torch.int32).to(self.device)
        K.kv_fork(self.k_rings, self.v_rings, index, self.positions)
        follow = [t for t in (self.tokens, self.logits, self.logprobs) if t is not None]
        if any(self._states[i] is not self._states[s] for i, s in enumerate(src)):
            follow += [self.w_up, self.w_gate, self.w_down]
        index = index.long()
        for t in follow:
            t.copy_(t.index_select(0, index))
        self.host_positions = [self.host_positions[s] for s in src]
        self._states = [self._states[s] for s in src]
        self._key = self._state_key(self._states)
