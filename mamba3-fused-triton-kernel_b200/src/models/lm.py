"""Token-by-token decoding of a ``MambaLMHeadModel``.

The reference has no decode path for its language model, only the
sequence ``forward`` (src/models/mamba3.py:473-481: embedding, blocks
``x + mixer(norm(x))`` each optionally followed by ``x + mlp(mlp_norm(x))``,
``norm_f``, ``lm_head``).  ``Mamba3LMDecoder.step`` computes the same thing
for one token per sequence with every mixer in its decode form:

    x = embedding(ids)
    xn = norm_0(x)
    for l:  o = mixer_l.step(xn)
            [MLP]  x, xm = x + o, mlp_norm_l(x + o);  x = x + mlp_l(xm)
            x, xn = x + o (or x), norm_{l+1}(x)      (norm_f after the last block)
    logits = lm_head(xn)

With a CUDA backend the residual add and the following norm are one kernel
(``m3_residual_rmsnorm``), every projection goes through
``src.kernels.linear.linear``, and ``warmup_cuda_graph`` captures the whole
token step -- embedding gather, all layers, the final norm and the LM head --
in one CUDA graph.

``generate`` decodes on from a prompt: after every token step the next token
of each row is chosen on the GPU (``src.kernels.logits.next_tokens``:
penalties for repeated tokens, a bias, a mask of allowed tokens, the largest
logit or a draw), and fed to the next step without the host waiting.  With
``w4_group_size`` every projection -- the layers', the MLPs' and the LM
head's -- is held in 4 bits (``src.kernels.linear_w4``).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from src.kernels.linear import linear
from src.kernels.linear_w4 import W4Projection
from src.kernels.logits import next_tokens
from src.kernels.norm import residual_rmsnorm
from src.models.inference import Mamba3Decoder, check_device_error


def _linear(model, name: str, i: int):
    """The model's LM head, or ``fc1`` / ``fc2`` of block ``i``'s MLP."""
    return model.lm_head if name == "lm_head" else getattr(model.mlp_layers[i], name)


class Mamba3LMDecoder:
    """Decoder over a ``MambaLMHeadModel``.  ``decoder_kwargs``: the
    ``Mamba3Decoder`` backend flags, applied to every layer;
    ``use_cuda_graph`` captures the whole token step; ``w4_group_size``
    (32, 64 or 128; full-fused backend) holds every projection in 4 bits."""

    def __init__(self, model, use_cuda_graph: bool = False, w4_group_size: int | None = None, **decoder_kwargs):
        self.model = model
        self.blocks = list(model.layers)
        if not self.blocks:
            raise ValueError("model has no layers")
        self.layers = [Mamba3Decoder(b.mixer, w4_group_size=w4_group_size, **decoder_kwargs) for b in self.blocks]
        first = self.layers[0]
        self.cuda = first.use_triton or first.use_triton_fused or first.use_triton_full_fused or \
            first.use_compile or first.use_compile_cuda_graph
        self.use_cuda_graph = bool(use_cuda_graph) and self.cuda
        self._graph = None
        self._graph_ids = None
        self._graph_logits = None
        self._graph_states = None
        self._w4 = None
        if w4_group_size is not None:
            places = [("lm_head", 0)] + [(fc, i) for i in range(len(model.mlp_layers or [])) for fc in ("fc1", "fc2")]
            self._w4 = {at: W4Projection(lambda at=at: _linear(model, *at).weight, w4_group_size) for at in places}

    def _weight(self, name: str, i: int = 0):
        """The weight of the LM head or of block ``i``'s MLP, or its 4-bit
        form."""
        return _linear(self.model, name, i).weight if self._w4 is None else self._w4[name, i].get()

    @property
    def vocab_size(self) -> int:
        return self.model.vocab_size

    def init_state(self, batch_size: int, device=None) -> list:
        """One ``{angle_state, ssm_state, bx_prev}`` dict per layer."""
        return [layer.init_state(batch_size, device=device) for layer in self.layers]

    def _norm_after(self, i: int):
        """The norm applied to the residual stream after block ``i``'s
        residual add: the next block's norm, or ``norm_f`` after the last."""
        return self.blocks[i + 1].norm if i + 1 < len(self.blocks) else self.model.norm_f

    def _step_eager(self, ids: torch.Tensor, states: list) -> torch.Tensor:
        m = self.model
        x = m.embedding(ids)
        mlp = m.mlp_layers
        if not self.cuda:
            xn = self.blocks[0].norm(x)
            for i, (layer, st) in enumerate(zip(self.layers, states)):
                o, _ = layer._step_pytorch(xn, st)
                x = x + o
                if mlp is not None:
                    x = x + mlp[i](m.mlp_norms[i](x))
                xn = self._norm_after(i)(x)
            return F.linear(xn, m.lm_head.weight)
        _, xn = residual_rmsnorm(x, None, self.blocks[0].norm.weight, self.blocks[0].norm.eps)
        for i, (layer, st) in enumerate(zip(self.layers, states)):
            o, _ = layer._graph_step_fn()(xn, st)
            if mlp is not None:
                x, xm = residual_rmsnorm(x, o, m.mlp_norms[i].weight, m.mlp_norms[i].eps)
                gate, val = linear(xm, self._weight("fc1", i)).chunk(2, dim=-1)
                o = linear((F.silu(gate) * val).contiguous(), self._weight("fc2", i))
            nrm = self._norm_after(i)
            x, xn = residual_rmsnorm(x, o, nrm.weight, nrm.eps)
        return linear(xn, self._weight("lm_head"))

    def warmup_cuda_graph(self, states: list, n_warmup: int = 3) -> None:
        """``n_warmup`` eager token steps (token id 0), then capture one token
        step in a CUDA graph that updates ``states`` in place."""
        if not self.use_cuda_graph:
            return
        h = states[0]["ssm_state"]
        self._graph_ids = torch.zeros(h.shape[0], dtype=torch.long, device=h.device)
        for _ in range(n_warmup):
            self._step_eager(self._graph_ids, states)
        torch.cuda.synchronize(h.device)
        self.check_device_error()
        self.update_w4()
        self._graph = torch.cuda.CUDAGraph()
        self._graph_states = states
        with torch.cuda.graph(self._graph):
            self._graph_logits = self._step_eager(self._graph_ids, states)

    def update_w4(self, force: bool = False) -> None:
        """Quantise the projections that have changed, in place: a captured
        step sees a changed weight after this (``Mamba3Decoder.update_w4``).
        Called by ``warmup_cuda_graph``, ``decode_sequence`` and
        ``generate``."""
        for layer in self.layers:
            layer.update_w4(force)
        for projection in (self._w4 or {}).values():
            projection.refresh() if force else projection.get()

    def check_device_error(self) -> None:
        """Raise if a library kernel gave up a bounded wait since the last
        check; logits, tokens and states since then are undefined
        (``Mamba3Decoder.check_device_error``).  Synchronises the device.
        Called by ``warmup_cuda_graph`` and at the end of ``decode_sequence``
        (not while it is captured) and ``generate``."""
        check_device_error(self.layers)

    def step(self, input_ids: torch.Tensor, states: list) -> tuple:
        """One token per sequence: ``input_ids`` (batch,) -> (logits
        (batch, vocab), states)."""
        if self._graph is not None:
            if states is not self._graph_states:
                raise ValueError("a captured decoder steps the states it was captured with")
            self._graph_ids.copy_(input_ids)
            self._graph.replay()
            return self._graph_logits, states
        return self._step_eager(input_ids, states), states

    def decode_sequence(self, input_ids: torch.Tensor, states: list | None = None) -> tuple:
        """Feed ``input_ids`` (batch, length) token by token; returns
        (logits (batch, length, vocab), states) -- the reference ``forward``'s
        output, computed by the decode step."""
        B, L = input_ids.shape
        if states is None:
            states = self.init_state(B, device=input_ids.device)
        outs = []
        if self._graph is not None:
            self.update_w4()
        with torch.no_grad():
            for t in range(L):
                logits, states = self.step(input_ids[:, t], states)
                outs.append(logits.clone())
        if self.cuda and L > 0 and not (input_ids.is_cuda and torch.cuda.is_current_stream_capturing()):
            self.check_device_error()
        return torch.stack(outs, dim=1), states

    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, *, prompt_lengths: torch.Tensor | None = None,
                 states: list | None = None, eos_token_id: int | None = None, temperature=None,
                 seeds: torch.Tensor | None = None, **adjust) -> tuple:
        """Continue ``input_ids`` (batch, length) by up to ``max_new_tokens``
        a row; returns (tokens (batch, length + max_new_tokens) int64,
        logprobs of the same shape, lengths (batch,)).

        prompt_lengths  (batch,): rows with a shorter prompt, padded on the
                 right; each goes on behind its own last token
        states   a decode state to start from (a captured decoder: the one it
                 was captured with); without it a new one, or the captured
                 one set to zero
        eos_token_id  a row that has produced it stops
        temperature, seeds  as in ``next_tokens``; the draw of a token uses
                 its place in the row as the position
        adjust   ``next_tokens``' penalties, ``bias`` and ``allowed``; the
                 prompt counts as seen, not as generated

        ``lengths`` counts a row's prompt and what it produced (its
        ``eos_token_id`` with it); places behind that hold 0, as do the
        logprobs of the prompt.  Only the model's own vocabulary is produced,
        not what pads it.  Waits for the GPU once at the end, to raise if a
        kernel gave up (``check_device_error``).  Needs a CUDA backend."""
        if not self.cuda:
            raise RuntimeError("generate needs a CUDA backend")
        assert input_ids.is_cuda and input_ids.dim() == 2 and input_ids.shape[1] > 0, \
            "input_ids must be a (batch, length) CUDA tensor"
        assert max_new_tokens >= 0
        B, L = input_ids.shape
        dev = input_ids.device
        vocab = self.model.config.vocab_size
        if prompt_lengths is None:
            prompt = torch.full((B,), L, dtype=torch.long, device=dev)
        else:
            assert prompt_lengths.shape == (B,) and not prompt_lengths.is_floating_point()
            prompt = prompt_lengths.to(device=dev, dtype=torch.long)
        total = L + max_new_tokens
        tokens = torch.zeros(B, total, dtype=torch.long, device=dev)
        place = torch.arange(L, device=dev)
        tokens[:, :L] = torch.where(place < prompt[:, None], input_ids.long(), 0)
        logprobs = torch.zeros(B, total, dtype=torch.float32, device=dev)
        if B == 0:
            return tokens, logprobs, prompt
        # one look at the inputs, before the GPU sees them as indices
        low, high, short, long = (int(v) for v in torch.stack(
            (tokens.min(), tokens.max(), prompt.min(), prompt.max())).tolist())
        if low < 0 or high >= vocab:
            raise ValueError(f"input_ids must be in [0, {vocab})")
        if short < 1 or long > L:
            raise ValueError(f"prompt_lengths must be in [1, {L}]")
        if eos_token_id is not None and not 0 <= eos_token_id < vocab:
            raise ValueError(f"eos_token_id must be in [0, {vocab})")
        assert temperature is None or seeds is not None, "a temperature needs seeds"
        given = states if states is not None else self._graph_states
        if given is not None and given[0]["ssm_state"].shape[0] != B:
            raise ValueError(f"the states hold {given[0]['ssm_state'].shape[0]} rows, input_ids {B}")
        if states is None:
            if self._graph is not None:
                states = self._graph_states
                for st in states:
                    for v in st.values():
                        v.zero_()
            else:
                states = self.init_state(B, device=dev)
        if self._graph is not None:
            self.update_w4()
        end = prompt + max_new_tokens
        lengths = prompt.clone()
        going = torch.ones(B, dtype=torch.bool, device=dev)
        seen = torch.empty(B, dtype=torch.long, device=dev)
        with torch.no_grad():
            for t in range(total - 1):
                logits, states = self.step(tokens[:, t], states)
                if t + 1 < short:
                    continue
                seen.fill_(t + 1)
                ids, lp = next_tokens(logits[:, :vocab], tokens, seen, prompt, temperature=temperature, seeds=seeds,
                                      positions=seen if temperature is not None else None, **adjust)
                write = going & (prompt <= t + 1) & (t + 1 < end)
                tokens[:, t + 1] = torch.where(write, ids, tokens[:, t + 1])
                logprobs[:, t + 1] = torch.where(write, lp, 0.0)
                lengths += write
                if eos_token_id is not None:
                    going &= ~(write & (ids == eos_token_id))
        self.check_device_error()
        return tokens, logprobs, lengths
