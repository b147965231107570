"""One decode step of a patched model as a CUDA graph, replayed once per token.

Eager decoding of a patched model is bound by the interpreter, not by the GPU: a decoder block is
eleven kernels of a few microseconds each, and Python needs about 25 microseconds to issue one.  The
reference does not meet this problem (MLX evaluates a lazily built graph); here the equivalent is a
captured CUDA graph.  Every kernel of the patched decode step takes what changes from token to token
from device memory -- the token ids, the cache's per-sequence lengths (incremented on the device), the
cache rows themselves -- so one capture serves every later token.

    decoder = GraphedDecoder(model, batch=1, capacity=4096)       # inside apply_metile_to_torch_lm(...)
    logits = decoder.prefill(prompt_tokens)                       # eager
    tokens = decoder.generate(logits.argmax(-1), steps=128)       # graph replays, no host sync between

The model must offer `make_cache(batch, capacity)` returning `blocks.KVCache` objects and must run its
decode step through the patched path (the `attention` feature on, INT4 projections): a module that
falls back to its own forward slices the cache at the host's count, which a graph would freeze.
"""

from __future__ import annotations

import inspect

import torch

from .. import backends


def _logits_of(output):
    return getattr(output, "logits", output)


def _takes(function, parameter):
    try:
        return parameter in inspect.signature(function).parameters
    except (TypeError, ValueError):  # not every callable tells
        return False


class GraphedDecoder:
    def __init__(self, model, batch=1, capacity=4096):
        self.model = model
        self.batch, self.capacity = int(batch), int(capacity)
        self.cache = model.make_cache(self.batch, self.capacity)
        device = self.cache[0].keys.device
        self.device = device
        self._keeps_logits = _takes(model.forward, "logits_to_keep")
        self.token = torch.zeros((self.batch, 1), dtype=torch.long, device=device)   # input of the next step
        self.logits = None                                                          # output of the last step
        self.graph = None
        self.stream = torch.cuda.Stream(device)

    # ------------------------------------------------------------------------------------------
    def prefill(self, tokens):
        """Run the prompt [batch, length] eagerly through the model's own prefill path; returns the
        last position's logits [batch, vocabulary] (float32)."""
        if tokens.shape[0] != self.batch or tokens.shape[1] >= self.capacity:
            raise ValueError("prompt does not fit the decoder's batch or capacity")
        for cache in self.cache:
            cache.reset(0)
        # Only the last position's logits are asked for: a head over the whole prompt is most of a small model.
        last_only = {"logits_to_keep": 1} if self._keeps_logits else {}
        with torch.no_grad():
            out = _logits_of(self.model(tokens, cache=self.cache, **last_only))
        return out[:, -1, :].float()

    def _step(self):
        out = _logits_of(self.model(self.token, cache=self.cache))
        # The next step's input is chosen on the device: replays need no host in between.
        return backends.greedy_token(out[:, -1, :], self.token)

    def _capture(self):
        """Warm every lazily built piece on scratch caches, then capture one step on the real ones."""
        lengths = [cache.length for cache in self.cache]
        if min(lengths) < 1:
            raise ValueError("prefill before the first decode step")
        real, token = self.cache, self.token.clone()
        # Inside the `with` the current stream IS self.stream: what the caller queued before must be waited
        # for here, outside it.
        self.stream.wait_stream(torch.cuda.current_stream(self.device))
        with torch.no_grad(), torch.cuda.stream(self.stream):
            scratch = self.model.make_cache(self.batch, self.capacity)
            for cache, length in zip(scratch, lengths):
                cache.reset(length)
            self.cache = scratch
            self._step()                      # builds executors and fused q|k|v triples
            self.cache = real
            self.token.copy_(token)
            self.stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=self.stream):
                self.logits = self._step()
            for cache, length in zip(self.cache, lengths):   # capture ran the host-side bookkeeping once
                cache.length = length
        torch.cuda.current_stream(self.device).wait_stream(self.stream)
        self.graph = graph

    def step(self, token=None):
        """One decode step.  `token` [batch] (long) overrides the device-side choice of the previous
        step.  Returns the logits buffer [batch, vocabulary] (overwritten by the next step)."""
        if token is not None:
            self.token.copy_(token.reshape(self.batch, 1))
        if self.graph is None:
            self._capture()
        if self.cache[0].length + 1 > self.capacity:
            raise ValueError("KV cache capacity exceeded")
        caller = torch.cuda.current_stream(self.device)
        self.stream.wait_stream(caller)       # the token and the caches as the caller's stream leaves them
        with torch.cuda.stream(self.stream):
            self.graph.replay()
        caller.wait_stream(self.stream)
        for cache in self.cache:
            cache.length += 1                 # the device-side count was advanced by the graph
        return self.logits

    def generate(self, first_token, steps):
        """Greedy decoding: `steps` graph replays fed by the device-side argmax; returns the generated
        tokens [batch, steps + 1] starting with `first_token`."""
        generated = [first_token.reshape(self.batch, 1).clone()]
        self.token.copy_(generated[0])
        for _ in range(steps):
            self.step()
            generated.append(self.token.clone())
        return torch.cat(generated, dim=1)


class GraphedBeamDecoder:
    """Beam search for a batch of requests over a paged cache, a step at a time as a replayed CUDA graph.

    The beams of a request share the pages of its prompt and of every page that was full when they parted, so a step
    copies at most the page in work of the beams that were dropped, whatever the length.  A step takes its pages, runs the
    model, selects and reorders on the device.  With one beam it is greedy decoding of requests of different lengths.
    Pages are not counted by who refers to them: every beam takes a page whenever it fills one, and those of dropped beams
    come back with the next prompts, so a pool of batch * beams * ceil(capacity / page_size) pages (the default) never runs out
    and a smaller one may.  A search takes all its steps, also when every beam has finished.

        decoder = GraphedBeamDecoder(model, batch=2, beams=4, capacity=4096)
        tokens, scores = decoder.search([first_prompt, second_prompt], steps=64)

    The model must offer `make_paged_cache` (blocks.TinyCausalLM does)."""

    def __init__(self, model, batch=1, beams=4, capacity=4096, page_size=16, pages=None, end_token=None):
        self.model, self.batch, self.beams, self.end_token = model, int(batch), int(beams), end_token
        if not 1 <= self.beams <= backends.MAX_BEAMS:
            raise ValueError(f"a search has from 1 to {backends.MAX_BEAMS} beams")
        rows, width = self.batch * self.beams, -(-capacity // page_size)
        self.cache = model.make_paged_cache(rows, rows * width if pages is None else pages, page_size, capacity)
        self.tables = self.cache[0].tables
        device = self.device = self.tables.lengths.device
        self.token = torch.zeros((rows, 1), dtype=torch.long, device=device)      # input of the next step
        self.scores = torch.zeros((self.batch, self.beams), dtype=torch.float32, device=device)
        self.finished = torch.zeros((self.batch, self.beams), dtype=torch.bool, device=device)
        self.parents = torch.zeros((self.batch, self.beams), dtype=torch.int32, device=device)
        self.graph = None
        self.stream = torch.cuda.Stream(device)
        self._keeps_logits = _takes(model.forward, "logits_to_keep")

    def _select(self, logits, scores, finished):
        selected = backends.beam_select(logits, scores, keep=self.beams,
                                        finished=None if self.end_token is None else finished, end_token=self.end_token)
        for kept, new in zip((self.scores, self.parents, self.token, self.finished), selected):
            kept.copy_(new.view(kept.shape))

    def _step(self):
        self.tables.grow()
        logits = _logits_of(self.model(self.token, cache=self.cache))
        self._select(logits[:, -1, :], self.scores, self.finished)
        self.tables.reorder(self.parents, self.cache)

    def prefill(self, prompts):
        """Read one prompt (a row of token ids) for every request and select the first beams."""
        if len(prompts) != self.batch:
            raise ValueError("one prompt for every request of the batch")
        if not all(prompt.numel() for prompt in prompts):
            raise ValueError("a prompt has no token")
        self.tables.reset()
        # Only the last position's logits are asked for: a head over the whole prompt is most of a small model.
        last_only = {"logits_to_keep": 1} if self._keeps_logits else {}
        logits = []
        with torch.no_grad():
            for index, prompt in enumerate(prompts):
                self.tables.grow([prompt.numel() if row == index * self.beams else 0 for row in range(self.tables.requests)])
                tokens = prompt.reshape(1, -1).to(self.device)
                logits.append(_logits_of(self.model(tokens, cache=self.cache, **last_only))[:, -1])
            self.tables.fork(self.beams, self.cache)
            # The beams are still one: the first of them offers the candidates.
            start = torch.full((self.batch, self.beams), -torch.inf, device=self.device)
            start[:, 0] = 0.0
            self.finished.zero_()
            self._select(torch.cat(logits).repeat_interleave(self.beams, dim=0), start, self.finished)

    def _capture(self):
        """Warm what is built lazily on a scratch cache, then capture one step on the real one.  What fails on the way leaves
        the decoder as it was."""
        real, tables = self.cache, self.tables
        state = (self.token, self.scores, self.parents, self.finished)
        kept, counts = [t.clone() for t in state], (list(tables.held), tables.free, list(tables.shared))
        caller = torch.cuda.current_stream(self.device)
        self.stream.wait_stream(caller)
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.no_grad(), torch.cuda.stream(self.stream):
                # A page for each request, and tables as wide as the real ones: their width decides what is launched.
                self.cache = self.model.make_paged_cache(tables.requests, tables.requests, tables.page_size, tables.capacity)
                self.tables = self.cache[0].tables
                try:
                    self._step()
                finally:
                    self.cache, self.tables = real, tables
                    for own, value in zip(state, kept):
                        own.copy_(value)
                    self.stream.synchronize()
                with torch.cuda.graph(graph, stream=self.stream):
                    self._step()
        finally:
            tables.held, tables.free, tables.shared = counts     # capture runs the host's bookkeeping once
            caller.wait_stream(self.stream)
        self.graph = graph

    def step(self):
        """One token for every beam; the decoder's token, scores, parents and finished are those of the new beams."""
        ones = [1] * self.tables.requests
        self.tables.fits(ones)
        if self.graph is None:
            self._capture()
        self.tables.account(ones)   # what the graph does on the device
        if self.beams > 1:
            self.tables.share()
        caller = torch.cuda.current_stream(self.device)
        self.stream.wait_stream(caller)
        with torch.cuda.stream(self.stream):
            self.graph.replay()
        caller.wait_stream(self.stream)

    def search(self, prompts, steps):
        """The `beams` best continuations by `steps` tokens found for every prompt: tokens [batch, beams, steps] and the sums
        of their log-probabilities [batch, beams], the best first.  A beam that has met the end token repeats it."""
        if steps < 1:
            raise ValueError("a search takes one step or more")
        self.prefill(prompts)
        tokens, parents = [self.token.clone()], []
        for _ in range(steps - 1):
            self.step()
            tokens.append(self.token.clone())
            parents.append(self.parents.clone())
        # Back along the parents, from the last selection to the first.
        at = torch.arange(self.beams, device=self.device).expand(self.batch, -1)
        out = []
        for index in range(steps - 1, -1, -1):
            out.append(torch.gather(tokens[index].view(self.batch, self.beams), 1, at))
            if index:
                at = torch.gather(parents[index - 1].long(), 1, at)
        return torch.stack(out[::-1], dim=2), self.scores.clone()
