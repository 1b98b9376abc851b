"""Residual block and language model with the interface of the reference's
``mamba3_ssm/block.py``: MambaBlock (:20-29), MLPBlock (:32-43) and MambaLMHeadModel
(:46-139: forward, allocate_inference_cache, step). Parameter names match, so
reference checkpoints load with ``load_state_dict``."""

from typing import List, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from .beam import beam_select, reorder_states_
from .config import MambaConfig
from .layer import Mamba3
from .losses import token_logprobs
from .ops import RMSNorm, argmax_rows, rmsnorm


class MambaBlock(nn.Module):
    """x + Mamba3(RMSNorm(x))."""

    def __init__(self, d_model: int, ssm_cfg: dict, device=None, dtype=None):
        super().__init__()
        self.norm = RMSNorm(d_model)
        self.mixer = Mamba3(d_model=d_model, **ssm_cfg, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.mixer(self.norm(x))


class MLPBlock(nn.Module):
    """SwiGLU feed-forward used when d_intermediate > 0 (plain PyTorch: not on the scan path)."""

    def __init__(self, d_model: int, d_intermediate: int, device=None, dtype=None):
        super().__init__()
        f = {"device": device, "dtype": dtype}
        self.fc1 = nn.Linear(d_model, 2 * d_intermediate, bias=False, **f)
        self.fc2 = nn.Linear(d_intermediate, d_model, bias=False, **f)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        gate, val = self.fc1(x).chunk(2, dim=-1)
        return self.fc2(F.silu(gate) * val)


class MambaLMHeadModel(nn.Module):
    """Embedding -> n_layer x MambaBlock [+ MLPBlock] -> RMSNorm -> LM head (tied)."""

    def __init__(self, config: MambaConfig, device=None, dtype=None):
        f = {"device": device, "dtype": dtype}
        super().__init__()
        self.config = config
        v = config.vocab_size
        r = v % config.pad_vocab_size_multiple
        if r:
            v += config.pad_vocab_size_multiple - r
        self.vocab_size = v
        self.embedding = nn.Embedding(v, config.d_model, **f)
        self.layers = nn.ModuleList([MambaBlock(config.d_model, config.ssm_cfg, **f) for _ in range(config.n_layer)])
        if config.d_intermediate > 0:
            self.mlp_norms = nn.ModuleList([RMSNorm(config.d_model) for _ in range(config.n_layer)])
            self.mlp_layers = nn.ModuleList([MLPBlock(config.d_model, config.d_intermediate, **f)
                                             for _ in range(config.n_layer)])
        else:
            self.mlp_norms = None
            self.mlp_layers = None
        self.norm_f = RMSNorm(config.d_model)
        self.lm_head = nn.Linear(config.d_model, v, bias=False, **f)
        if device is not None:
            for mod in [self.norm_f] + [blk.norm for blk in self.layers]:
                mod.weight = nn.Parameter(mod.weight.data.to(device))
        if config.tie_embeddings:
            self.lm_head.weight = self.embedding.weight

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        x = self.embedding(input_ids)
        for i, block in enumerate(self.layers):
            x = block(x)
            if self.mlp_layers is not None:
                x = x + self.mlp_layers[i](self.mlp_norms[i](x))
        return self.lm_head(self.norm_f(x))

    def token_logprobs(self, input_ids: torch.Tensor, mask: torch.Tensor = None,
                       temperature: float = 1.0) -> torch.Tensor:
        """log p(input_ids[:, t + 1] | input_ids[:, :t + 1]) in fp32, (B, L - 1), from the logits
        by losses.token_logprobs: what a policy, a reference model or an evaluation records
        of given answers. mask (B, L - 1), optional: positions with 0 give 0."""
        logits = self.forward(input_ids)[:, :-1]
        return token_logprobs(logits, input_ids[:, 1:], mask=mask, temperature=temperature)

    def allocate_inference_cache(self, batch_size: int) -> List[Tuple[torch.Tensor, ...]]:
        return [blk.mixer.allocate_inference_cache(batch_size) for blk in self.layers]

    def prefill(self, input_ids: torch.Tensor, cache=None):
        """Run a whole prompt (B, L) through the chunked scans and return (logits (B, L, V),
        cache), the decode cache after the last token (a list of (angle, ssm, bx_prev) per
        layer, as allocate_inference_cache lays it out), ready for step(). Continues from
        ``cache`` when given (chunked prefill of a long prompt). Not in the reference, whose
        generate loop prefills one step() per prompt token; the result is that of stepping
        through the prompt."""
        x = self.embedding(input_ids)
        new_cache = []
        for i, block in enumerate(self.layers):
            out, c = block.mixer(block.norm(x), cache=None if cache is None else cache[i], return_cache=True)
            x = x + out
            new_cache.append(c)
            if self.mlp_layers is not None:
                x = x + self.mlp_layers[i](self.mlp_norms[i](x))
        return self.lm_head(self.norm_f(x)), new_cache

    def _norms_after(self, i):
        """The norm that follows layer i's mixer residual add: the MLP norm of layer i,
        the next block's norm, or norm_f."""
        if self.mlp_layers is not None:
            return self.mlp_norms[i]
        return self.layers[i + 1].norm if i + 1 < len(self.layers) else self.norm_f

    def step(self, input_ids: torch.Tensor, cache: List[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]):
        if input_ids.dim() == 1:
            input_ids = input_ids.unsqueeze(-1)
        x = self.embedding(input_ids).squeeze(1)
        new_cache = []
        h = self.layers[0].norm(x) if self.layers else self.norm_f(x)
        for i, block in enumerate(self.layers):
            out, a, s, b = block.mixer.step(h, *cache[i])
            new_cache.append((a, s, b))
            # x = x + out, then the next norm, in one kernel
            nrm = self._norms_after(i)
            x_new = torch.empty_like(x)
            h = rmsnorm(x, nrm.weight, nrm.eps, residual=out, residual_out=x_new)
            x = x_new
            if self.mlp_layers is not None:
                nxt = self.layers[i + 1].norm if i + 1 < len(self.layers) else self.norm_f
                x_new = torch.empty_like(x)
                h = rmsnorm(x, nxt.weight, nxt.eps, residual=self.mlp_layers[i](h), residual_out=x_new)
                x = x_new
        return self.lm_head(h), new_cache

    # ------------------------------------------------------------------------------
    def decode_graph(self, batch_size: int, greedy: bool = True) -> "DecodeGraph":
        """A CUDA-graph decode loop for this model at a fixed batch size (see DecodeGraph).
        Not part of the reference interface; step() keeps the reference's semantics."""
        return DecodeGraph(self, batch_size, greedy)

    def beam_graph(self, batch_size: int, num_beams: int, end_token: int = None) -> "BeamGraph":
        """A CUDA-graph beam search for this model at a fixed number of prompts and beams (see
        BeamGraph). Not part of the reference interface."""
        return BeamGraph(self, batch_size, num_beams, end_token)

    def beam_search(self, input_ids: torch.Tensor, num_beams: int, max_new_tokens: int, end_token: int = None,
                    length_penalty: float = 0.0):
        """The num_beams best continuations of each prompt (B, L): (tokens (B, num_beams, n), scores
        (B, num_beams)), the best first; see BeamGraph.search. Captures a graph for this one
        search: keep a ``beam_graph`` for several."""
        graph = self.beam_graph(input_ids.shape[0], num_beams, end_token)
        return graph.search(input_ids, max_new_tokens, length_penalty)


class _StepGraph:
    """One whole decode step (embedding, every layer's norm / in_proj / fused step kernel / out_proj /
    residual, norm_f, lm_head and, with ``greedy``, the argmax) as one CUDA graph over static
    tensors: the decode cache, updated in place, ``tokens`` and ``logits``."""

    def __init__(self, model: "MambaLMHeadModel", batch_size: int, greedy: bool = True):
        dev = model.embedding.weight.device
        if dev.type != "cuda":
            raise RuntimeError("DecodeGraph needs the model on a CUDA device")
        self.model = model
        self.greedy = greedy
        self.tokens = torch.zeros(batch_size, dtype=torch.long, device=dev)
        self.cache = model.allocate_inference_cache(batch_size)
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side), torch.no_grad():
            for _ in range(2):  # warm the caching allocator and the libraries outside the graph
                self._body()
        torch.cuda.current_stream(dev).wait_stream(side)
        self.reset()
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(self.graph, capture_error_mode="relaxed"):
            self.logits = self._body()
        self.reset()

    def _body(self):
        m = self.model
        x = m.embedding(self.tokens)
        h = m.layers[0].norm(x) if m.layers else m.norm_f(x)
        for i, blk in enumerate(m.layers):
            out = blk.mixer.step_inplace(h, *self.cache[i])
            nrm = m._norms_after(i)
            h = rmsnorm(x, nrm.weight, nrm.eps, residual=out, residual_out=x)  # x += out; norm
            if m.mlp_layers is not None:
                nxt = m.layers[i + 1].norm if i + 1 < len(m.layers) else m.norm_f
                h = rmsnorm(x, nxt.weight, nxt.eps, residual=m.mlp_layers[i](h), residual_out=x)
        logits = m.lm_head(h)
        if self.greedy:
            argmax_rows(logits, out=self.tokens)
        return logits

    def reset(self):
        for a, s, b in self.cache:
            a.zero_()
            s.zero_()
            b.zero_()


class DecodeGraph(_StepGraph):
    """Replays one whole decode step (embedding, every layer's norm / in_proj / fused step
    kernel / out_proj / residual, norm_f, lm_head and, with ``greedy``, the argmax) as one
    CUDA graph. The decode cache lives in static tensors updated in place; ``logits`` and
    ``tokens`` are static buffers overwritten by every call.

        g = model.decode_graph(batch)          # captures on the current device
        g.prefill(prompt)                      # whole prompt through the chunked scans
        for _ in range(n): tok = g.next()      # greedy: the argmax becomes the next input
    (``g.reset()`` then ``g.feed(t)`` per prompt token also works, like step().)
    """

    def prefill(self, prompt: torch.Tensor) -> torch.Tensor:
        """Replace the cache by that of the prompt (B, L), computed by MambaLMHeadModel.prefill
        (chunked scans, not one replay per token), and return the last position's logits
        (B, V); with ``greedy`` the next input token is their argmax."""
        with torch.no_grad():
            logits, cache = self.model.prefill(prompt.reshape(self.tokens.shape[0], -1))
            for dst, src in zip(self.cache, cache):
                for d, s_ in zip(dst, src):
                    d.copy_(s_)
            last = logits[:, -1]
            if self.greedy:
                argmax_rows(last, out=self.tokens)
        return last

    def feed(self, tokens: torch.Tensor) -> torch.Tensor:
        """One step on the given tokens (B,) or (B, 1); returns the static logits."""
        self.tokens.copy_(tokens.reshape(-1))
        self.graph.replay()
        return self.logits

    def next(self) -> torch.Tensor:
        """One greedy step on the previous step's argmax; returns the static token buffer."""
        self.graph.replay()
        return self.tokens


class BeamGraph(_StepGraph):
    """Beam search with one CUDA graph a token: the selection among the previous step's logits
    (beam.beam_select), the beams' states moved to the beams that continue them
    (beam.reorder_states_, in place), and the decode step of DecodeGraph for batch_size * num_beams
    rows. The tokens come from the selection, so there is no feeding of single ones.

        g = model.beam_graph(batch, beams, end_token)
        tokens, scores = g.search(prompt, max_new_tokens)
    """

    def __init__(self, model: "MambaLMHeadModel", batch_size: int, num_beams: int, end_token: int = None):
        dev = model.embedding.weight.device
        if dev.type != "cuda":
            raise RuntimeError("BeamGraph needs the model on a CUDA device")
        self.vocabulary = min(model.config.vocab_size, model.vocab_size)  # without the padding of the weights
        if end_token is not None and not 0 <= end_token < self.vocabulary:
            raise ValueError(f"BeamGraph: end_token {end_token} is outside the vocabulary of {self.vocabulary}")
        if batch_size < 1 or not 1 <= num_beams <= 32:
            raise ValueError(f"BeamGraph: at least one prompt and 1 to 32 beams, got {batch_size} and {num_beams}")
        self.end_token = end_token
        shape = (batch_size, num_beams)
        self.ahead = torch.zeros(*shape, model.vocab_size, dtype=model.lm_head.weight.dtype, device=dev)
        self.scores = torch.zeros(shape, dtype=torch.float32, device=dev)
        self.parents = torch.zeros(shape, dtype=torch.int64, device=dev)
        self.finished = torch.zeros(shape, dtype=torch.bool, device=dev)
        super().__init__(model, batch_size * num_beams, greedy=False)

    def _body(self):
        ended = self.end_token is not None
        sel = beam_select(self.ahead[..., :self.vocabulary], self.scores, finished=self.finished if ended else None,
                          end_token=self.end_token if ended else 0)
        self.scores.copy_(sel.scores)
        self.parents.copy_(sel.parents)
        self.tokens.copy_(sel.tokens.view(-1))
        if ended:
            self.finished.copy_(self.finished.gather(1, sel.parents) | (sel.tokens == self.end_token))
        reorder_states_(self.cache, self.parents)
        logits = super()._body()
        self.ahead.copy_(logits.view_as(self.ahead))
        return logits

    def reset(self):
        """As before any search."""
        super().reset()
        for t in (self.ahead, self.scores, self.parents, self.finished, self.tokens):
            t.zero_()

    @torch.no_grad()
    def search(self, prompt: torch.Tensor, max_new_tokens: int, length_penalty: float = 0.0):
        """(tokens (B, num_beams, n), scores (B, num_beams)) for prompts (B, L), n <= max_new_tokens, the
        best first. scores: the sum of the tokens' log-probabilities over their number (up to the
        end token, which counts) to the power of length_penalty. Behind the end token a row is filled
        with it; the search ends early once every beam has ended (looked at every 16 tokens)."""
        b, k = self.scores.shape
        if prompt.dim() != 2 or prompt.shape[0] != b or prompt.shape[1] == 0:
            raise ValueError(f"BeamGraph: prompts ({b}, length) expected, got {tuple(prompt.shape)}")
        if max_new_tokens < 1:
            raise ValueError(f"BeamGraph: max_new_tokens must be 1 or more, got {max_new_tokens}")
        dev = self.scores.device
        logits, cache = self.model.prefill(prompt)
        # every beam starts from the prompt; all but the first are empty places, so that the first step takes its best tokens
        reorder_states_(cache, torch.zeros((b, k), dtype=torch.int64, device=dev), out=self.cache)
        self.ahead.copy_(logits[:, -1:].expand(b, k, logits.shape[-1]))
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0.0
        self.finished.zero_()
        parents = torch.empty((max_new_tokens, b, k), dtype=torch.int64, device=dev)
        tokens = torch.empty_like(parents)
        n = 0
        while n < max_new_tokens:
            self.graph.replay()
            parents[n].copy_(self.parents)
            tokens[n].copy_(self.tokens.view(b, k))
            n += 1
            if self.end_token is not None and n % 16 == 0 and bool(self.finished.all()):
                break
        # from the last tokens back through the beams that they continue
        at = torch.arange(k, device=dev).expand(b, k)
        out = torch.empty((b, k, n), dtype=torch.int64, device=dev)
        for t in range(n - 1, -1, -1):
            out[:, :, t] = tokens[t].gather(1, at)
            at = parents[t].gather(1, at)
        scores = self.scores
        if length_penalty:
            length = n if self.end_token is None else ((out == self.end_token).cumsum(-1) == 0).sum(-1).add(1).clamp(max=n)
            scores = scores / (length ** length_penalty if isinstance(length, int) else length.float() ** length_penalty)
        best, order = scores.sort(dim=1, descending=True, stable=True)
        return out.gather(1, order.unsqueeze(-1).expand_as(out)), best
