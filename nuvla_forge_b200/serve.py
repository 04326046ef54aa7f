"""Serving: planning with the DiT sampling loop in one CUDA graph, and answering token by token.

At serving batch sizes the sampler is launch-bound: every Euler step runs the
whole DiT (a few hundred small kernels) on a [B, horizon] trajectory. The
``GraphedPlanner`` captures all ``steps`` Euler steps for a fixed batch size
and context length once (after a warm-up on a side stream, which also
initialises every kernel's lazily created state), and then serves each
request with two copies into static buffers and one graph replay.

    planner = GraphedPlanner(model, batch_size=8, context_len=L, steps=10)
    waypoints = planner(context)          # context: model.context(images, text_tokens)

``ReasoningDecoder`` answers with the reasoning head: the prompt (images and instruction) fills a
paged key-value cache, then one captured graph per token appends to it, attends over it and scores
the next token.

    decoder = ReasoningDecoder(model, batch_size=8, prompt_len=64, max_new=256)
    answer = decoder(images, text_tokens)   # tokens, log probabilities, entropy, alternatives, states
    waypoints = planner(answer.states)      # the DiT attends to the answer's states too
    waypoints = model.dit.sample(answer.context(b))   # or to one answer's, cut behind its stop token

On CPU (or with ``graph=False``) both run the same code eagerly; so does a ``ReasoningDecoder`` of a model
with ``fused=False`` or without native kernels, whose reference operators read indices back.
The reference has no inference path beyond ``TrajectoryDiT.sample``
(nuvla_forge/model/dit.py:221-230, never called in its repository).
"""

from __future__ import annotations

import threading
from typing import NamedTuple

import torch

from . import _native as nat
from .models.nuvla import NuVLA
from .ops import paged, token_logprobs


class GraphedPlanner:
    def __init__(self, model: NuVLA, batch_size: int, context_len: int, steps: int = 10, graph: bool = True,
                 warmup: int = 2):
        self.model = model
        self.dit = model.dit
        self.steps = steps
        p = next(model.parameters())
        self.device = p.device
        d_ctx = self._context_dim(model)
        self.ctx = torch.zeros(batch_size, context_len, d_ctx, device=self.device, dtype=p.dtype)
        self.z0 = torch.zeros(batch_size, self.dit.horizon, self.dit.traj_dim, device=self.device)
        self.out = None
        self.graph = None
        if graph and self.device.type == "cuda":
            side = torch.cuda.Stream(self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side), torch.no_grad():
                for _ in range(warmup):
                    self.dit.sample(self.ctx, self.steps, z0=self.z0)
            torch.cuda.current_stream(self.device).wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g), torch.no_grad():
                self.out = self.dit.sample(self.ctx, self.steps, z0=self.z0)
            self.graph = g

    @staticmethod
    def _context_dim(model: NuVLA) -> int:
        cfg = model.cfg
        return cfg.t_dim if cfg.backbone_over_images else cfg.vision_dim

    @torch.no_grad()
    def __call__(self, context: torch.Tensor, z0: torch.Tensor | None = None) -> torch.Tensor:
        """Waypoints [B, horizon, traj_dim] for ``context`` [B, context_len, D] (fresh noise unless ``z0``)."""
        if context.shape != self.ctx.shape:
            raise ValueError(f"planner was built for context {tuple(self.ctx.shape)}, got {tuple(context.shape)}")
        self.ctx.copy_(context)
        if z0 is not None:
            self.z0.copy_(z0)
        else:
            self.z0.normal_()
        if self.graph is None:
            return self.dit.sample(self.ctx, self.steps, z0=self.z0)
        self.graph.replay()
        return self.out.clone()


class Answer(NamedTuple):
    tokens: torch.Tensor         # [B, max_new] int64
    logprobs: torch.Tensor       # [B, max_new] fp32, of the tokens (behind a stop token all scores are 0)
    entropy: torch.Tensor        # [B, max_new] fp32, of each token's distribution
    top_tokens: torch.Tensor     # [B, max_new, top_k] int64 (behind a stop token that token)
    top_logprobs: torch.Tensor   # [B, max_new, top_k] fp32
    lengths: torch.Tensor        # [B] int64, tokens up to and with the stop token
    states: torch.Tensor         # [B, prompt states + max_new, D], for the DiT's cross-attention: those of
                                 # ``model.context`` over instruction and ``tokens``, repeated stop tokens too

    def context(self, b: int) -> torch.Tensor:
        """States [1, n, D] of sequence ``b`` up to and with its stop token (waits for its length). The DiT attends to
        every state that it is given, so a plan from these does not depend on ``max_new``, one from ``states`` does."""
        n = self.states.shape[1] - self.tokens.shape[1] + int(self.lengths[b])
        return self.states[b, None, :n]


class ReasoningDecoder:
    """Greedy answers of the reasoning head over a paged key-value cache (causal backbone layout).

    Built for a batch size, ``prompt_len`` instruction tokens and ``max_new`` answer tokens (at most
    the model's text positions together). ``stop_token`` ends a sequence: its later tokens repeat it and
    score 0 (they are read like others, so that ``states`` are those of the returned tokens). A decoder
    works on one answer at a time: calls from several threads or streams wait for one another (build a
    decoder for each to have them at once). The reference has no decoding path.
    """

    @torch.inference_mode(False)  # buffers that calls in any mode can write
    def __init__(self, model: NuVLA, batch_size: int, prompt_len: int, max_new: int | None = None, top_k: int = 5,
                 page_size: int = 64, stop_token: int | None = None, graph: bool = True, warmup: int = 2):
        cfg = model.cfg
        max_new = cfg.n_reasoning if max_new is None else max_new
        if prompt_len < 1 or max_new < 1 or prompt_len + max_new > cfg.text_len:
            raise ValueError(f"{prompt_len} instruction and {max_new} answer tokens do not fit the model's "
                             f"{cfg.text_len} text positions")
        if not 1 <= top_k <= 32:
            raise ValueError(f"top_k {top_k} is not in 1..32")
        self.model, self.batch_size, self.prompt_len, self.max_new = model, batch_size, prompt_len, max_new
        self.top_k, self.stop_token = top_k, stop_token
        self.n_prompt = cfg.n_images * cfg.pooled_tokens + prompt_len
        self.cache = model.new_cache(batch_size, self.n_prompt + max_new, page_size)
        dev = model.lm_head.device
        B, N = batch_size, max_new
        self.token = torch.zeros(B, dtype=torch.int64, device=dev)
        self.live = torch.ones(B, dtype=torch.int32, device=dev)
        self.index = torch.zeros(1, dtype=torch.int64, device=dev)       # of the token to be read
        self.tokens = torch.zeros((B, N + 1), dtype=torch.int64, device=dev)
        self.logprobs = torch.zeros((B, N + 1), dtype=torch.float32, device=dev)
        self.entropy = torch.zeros((B, N + 1), dtype=torch.float32, device=dev)
        self.top_tokens = torch.zeros((B, N + 1, top_k), dtype=torch.int64, device=dev)
        self.top_logprobs = torch.zeros((B, N + 1, top_k), dtype=torch.float32, device=dev)
        self.lengths = torch.zeros(B, dtype=torch.int64, device=dev)
        self.states = torch.zeros((B, self.n_prompt + N, model.cfg.t_dim), dtype=model.lm_head.dtype, device=dev)
        self.graph = None
        self._turn = threading.Lock()
        self._done: torch.cuda.Event | None = None   # the last use of the buffers above, on any stream
        if graph and dev.type == "cuda" and cfg.fused and nat.HAS_NATIVE and model.lm_head.dtype in nat.DT:
            with torch.cuda.device(dev):  # the capture is of the current device's stream
                side = torch.cuda.Stream(dev)
                side.wait_stream(torch.cuda.current_stream(dev))
                with torch.cuda.stream(side):
                    for _ in range(max(1, warmup)):  # (the status words are made outside of the capture)
                        self._restart()
                        self._step()
                torch.cuda.current_stream(dev).wait_stream(side)
                self._restart()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    self._step()
            self.graph = g
        if dev.type == "cuda":
            self._done = torch.cuda.Event()
            self._done.record(torch.cuda.current_stream(dev))

    def _restart(self) -> None:
        self.index.zero_()
        self.live.fill_(1)
        self.lengths.zero_()
        self.token.zero_()
        self.cache.lengths.fill_(self.n_prompt)

    @torch.no_grad()
    def _choose(self, h: torch.Tensor, at: torch.Tensor) -> None:
        """The most likely next token of states h [B, D], written with its scores to column ``at`` [1]."""
        r = token_logprobs(self.model.text_logits(h), top_k=self.top_k, force_reference=not self.model.cfg.fused)
        top, scores, entropy = r.top_tokens, r.top_logprobs, r.entropy
        if self.stop_token is not None:
            off = self.live == 0
            top = top.masked_fill(off[:, None], self.stop_token)
            scores, entropy = scores.masked_fill(off[:, None], 0.0), entropy.masked_fill(off, 0.0)
        self.token.copy_(top[:, 0])
        self.lengths.add_(self.live)
        self.tokens.index_copy_(1, at, top[:, :1])
        self.logprobs.index_copy_(1, at, scores[:, :1])
        self.entropy.index_copy_(1, at, entropy[:, None])
        self.top_tokens.index_copy_(1, at, top[:, None])
        self.top_logprobs.index_copy_(1, at, scores[:, None])

    @torch.no_grad()
    def _step(self) -> None:
        """Read the token that was chosen last, choose the next one."""
        if self.stop_token is not None:
            self.live.mul_((self.token != self.stop_token).to(torch.int32))
        h = self.model.read_token(self.token, self.index + self.prompt_len, self.cache)
        self.states.index_copy_(1, self.index + self.n_prompt, h)
        self.index.add_(1)
        self._choose(h[:, 0], self.index)

    @torch.no_grad()
    def __call__(self, images: torch.Tensor, text_tokens: torch.Tensor) -> Answer:
        if text_tokens.shape != (self.batch_size, self.prompt_len):
            raise ValueError(f"decoder was built for instructions {(self.batch_size, self.prompt_len)}, got "
                             f"{tuple(text_tokens.shape)}")
        with self._turn, nat.on_device(self.token.device):  # (kernels launch on the current device)
            if self._done is None:
                return self._answer(images, text_tokens)
            stream = torch.cuda.current_stream(self.token.device)
            captured = torch.cuda.is_current_stream_capturing()  # (ordered by whoever replays it)
            if not captured:
                stream.wait_event(self._done)
            try:
                return self._answer(images, text_tokens)
            finally:
                if not captured:
                    self._done.record(stream)

    def _answer(self, images: torch.Tensor, text_tokens: torch.Tensor) -> Answer:
        h = self.model.read_prompt(images, text_tokens, self.cache)
        if h.shape[1] != self.n_prompt:
            raise ValueError(f"decoder was built for {self.n_prompt} prompt states, got {h.shape[1]}")
        self._restart()
        self.states[:, : self.n_prompt].copy_(h)
        self._choose(h[:, -1], self.index)
        for _ in range(self.max_new):
            if self.graph is not None:
                self.graph.replay()
            else:
                self._step()
        n = self.max_new
        return Answer(self.tokens[:, :n].clone(), self.logprobs[:, :n].clone(), self.entropy[:, :n].clone(),
                      self.top_tokens[:, :n].clone(), self.top_logprobs[:, :n].clone(),
                      self.lengths.clamp(max=n), self.states.clone())

    def check_status(self) -> None:
        """Raise if a kernel met an index out of range (synchronises)."""
        paged.check_status(self.token.device)
