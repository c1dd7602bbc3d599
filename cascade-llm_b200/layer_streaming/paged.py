"""Several sequences, or several sampled continuations of one prompt, over a
key-value cache in pages.

The reference decodes one request (``layer_streaming/llama31.py:34-54``, one
contiguous cache); this is an addition next to it. :class:`PagedKVCache` holds
the pages and their bookkeeping on the device; :class:`PagedBatchDecoder` runs
one token of every sequence per step with the weights resident in HBM:

=====================  ==========================================================
per layer              ``rmsnorm``, three ``gemm_bf16`` (q, k, v), ``paged_append``
                       (rotation and cache write), ``paged_attention``,
                       ``gemm_residual`` (o), ``rmsnorm``, ``gemm_swiglu``,
                       ``gemm_residual`` (down)
per step               ``pages_reserve`` (a page where a sequence needs one),
                       ``embedding``, the layers, ``rmsnorm``, ``gemm_bf16`` (head)
per token              ``sample``
between tokens         ``pages_fork``, ``pages_free``, ``pages_compact``
=====================  ==========================================================

Prompts run through the executor's own prefill; their keys and values are
copied into pages. Every step has fixed shapes and keeps lengths, tables and
free pages on the device, so it is captured once and replayed as a CUDA graph.
"""

import warnings

import torch

from . import _native, ops
from .llama31 import _SPLIT_K_MAX_TOKENS, _UNIT_OPS, _matrix_key

BF16 = torch.bfloat16


def _slots(values, device):
    return torch.as_tensor(values, dtype=torch.int32, device=device).reshape(-1)


class PagedKVCache:
    """Pages ``storage`` [layers, 2, pages, kv_heads, page_size, head_dim] and
    the device state of ``sequences`` slots: ``table`` (a slot's pages in order,
    -1 behind them), ``lengths`` and ``ref`` (table entries per page, 0 = free).

    Free pages are taken lowest index first. ``fork`` and ``reserve`` are all or
    nothing; their outcome stays in ``status`` on the device until
    :meth:`check` reads it (a synchronisation), so that steps need none.
    """

    def __init__(self, sequences, pages, max_length, layer_count=32, kv_heads=8, page_size=16, head_dim=128,
                 device="cuda:0", dtype=BF16):
        for name, value in (("sequences", sequences), ("pages", pages), ("max_length", max_length),
                            ("layer_count", layer_count), ("kv_heads", kv_heads), ("page_size", page_size)):
            if int(value) < 1:
                raise ValueError("{} must be positive".format(name))
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("the paged cache needs a CUDA device (there is no CPU path)")
        self.page_size = int(page_size)
        width = -(-int(max_length) // self.page_size)
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=self.device)  # noqa: E731
        # zeros: what nobody has written is then the same in every cache (torch.empty gives a NaN at times)
        self.storage = torch.zeros((layer_count, 2, pages, kv_heads, page_size, head_dim), dtype=dtype,
                                   device=self.device)
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=self.device)
        self.lengths, self.ref, self.status = ints(sequences), ints(pages), ints(1)
        self.workspace = ints(ops.pages_workspace_ints(pages))
        self._worst = ints(1)  # largest status since the last check (-1 counts as the largest)

    @property
    def max_length(self):
        return self.table.shape[1] * self.page_size

    def layer(self, index):
        """One layer's (k_pages, v_pages)."""

        return self.storage[index, 0], self.storage[index, 1]

    def _note(self):
        # as unsigned: -1 is above every count of missing pages
        worst, now = self._worst, self.status
        worst.copy_(torch.where(now < 0, now, torch.where(worst < 0, worst, torch.maximum(worst, now))))

    def reserve(self, extra):
        """lengths += extra (int32 per slot, on the device) with the pages that takes."""

        ops.pages_reserve(extra, self.table, self.lengths, self.ref, self.page_size, self.status, self.workspace)
        self._note()

    def fork(self, parents, children):
        """Empty slots `children` become copies of `parents`, pairwise."""

        ops.pages_fork(_slots(parents, self.device), _slots(children, self.device), self.table, self.lengths, self.ref,
                       self.storage, self.status, self.workspace)
        self._note()

    def free(self, slots):
        ops.pages_free(_slots(slots, self.device), self.table, self.lengths, self.ref)

    def compact(self):
        """Move the live pages into the pool's dense prefix; the number of live
        pages, on the device."""

        live = torch.empty(1, dtype=torch.int32, device=self.device)
        ops.pages_compact(self.table, self.ref, self.storage, self.table, self.ref, live, self.workspace)
        return live

    def check(self):
        """Raise if a reserve or a fork since the last check was refused."""

        worst = int(self._worst.item())
        self._worst.zero_()
        if worst > 0:
            raise RuntimeError("the paged cache is full: {} pages missing".format(worst))
        if worst < 0:
            raise ValueError("paged cache: wrong slots, or a sequence beyond max_length")


class PagedBatchDecoder:
    """One token of every slot per step.

    ``executor`` (a Llama31DecodeExecutor with the vocabulary resident) and
    ``runtime`` (``weights="hbm"``) supply the weights and run the prompts; the
    executor's own request is given up while a prompt is added. Slots that are
    empty take part as padding.
    """

    def __init__(self, executor, runtime, sequences, pages, max_length, page_size=16, use_graphs=True):
        if runtime.weights != "hbm":
            raise ValueError("the paged decoder needs HBM-resident weights (weights='hbm')")
        if executor.vocab_runtime is not None:
            raise ValueError("the paged decoder needs the vocabulary resident")
        if executor.decode_weights != "bf16":
            warnings.warn("decode_weights={!r} is for the executor's own one-token steps: the paged steps read the "
                          "bf16 weights".format(executor.decode_weights), stacklevel=2)
        self.executor, self.runtime, self.device = executor, runtime, executor.device
        self.sequences = int(sequences)
        self.cache = PagedKVCache(sequences, pages, max_length, executor.config.num_hidden_layers,
                                  page_size=page_size, device=self.device)
        self.use_graphs = bool(use_graphs)
        rows = self.sequences
        with torch.cuda.device(self.device):
            new = lambda width, dtype=BF16: torch.empty((rows, width), dtype=dtype, device=self.device)  # noqa: E731
            self._x, self._xn, self._q, self._attn = new(4096), new(4096), new(4096), new(4096)
            self._k, self._v, self._mlp = new(1024), new(1024), new(14336)
            self.logits = new(executor.config.vocab_size)
            self.tokens = torch.zeros(rows, dtype=torch.int64, device=self.device)
            self.logprobs = torch.zeros(rows, dtype=torch.float32, device=self.device)
            self._picked = torch.empty(rows, dtype=torch.int64, device=self.device)
            self._no_choice = torch.zeros(rows, dtype=torch.bool, device=self.device)  # since the last check
            self._full = torch.zeros(rows, dtype=torch.bool, device=self.device)  # the same
            self._position = torch.empty(rows, dtype=torch.int32, device=self.device)
            self._extra = torch.empty(rows, dtype=torch.int32, device=self.device)
            self._attention_ws = torch.zeros(ops.paged_attention_workspace_bytes(), dtype=torch.uint8,
                                             device=self.device)
        self._graph = None

    # ---------------------------------------------------------------- prompts
    def add(self, prompt_ids, slot):
        """Run a prompt (int64 [1, n]) and keep it in an empty slot; returns the
        logits behind its last token, fp32 [vocab]. If it fails, the slot stays
        empty; an earlier refused fork or step that nobody has read is raised
        before anything is taken."""

        if not 0 <= int(slot) < self.sequences:
            raise ValueError("slot {} is not one of {}".format(slot, self.sequences))
        if prompt_ids.dim() != 2 or prompt_ids.shape[0] != 1 or prompt_ids.shape[1] < 1:
            raise ValueError("a prompt must be [1, tokens] (got {})".format(list(prompt_ids.shape)))
        ex, cache = self.executor, self.cache
        if int(cache.lengths[slot]):
            raise ValueError("slot {} is in use".format(slot))
        length = int(prompt_ids.shape[1])
        if length > cache.max_length:
            raise ValueError("a prompt of {} tokens passes max_length={}".format(length, cache.max_length))
        with torch.cuda.device(self.device), torch.inference_mode():
            cache.check()
            extra = torch.zeros(self.sequences, dtype=torch.int32, device=self.device)
            extra[slot] = length
            cache.reserve(extra)
            cache.check()
            try:
                ex.kv_cache.clear()
                state = ex.finish(self.runtime.run(ex, ex.begin(prompt_ids)))
                position = torch.arange(length, dtype=torch.int32, device=self.device)
                sequence = torch.full((length,), int(slot), dtype=torch.int32, device=self.device)
                for layer in range(ex.config.num_hidden_layers):
                    # the executor's keys are rotated already: [heads, n, dim] read as tokens
                    key, value = (part[:, :length].transpose(0, 1) for part in (ex.kv_cache.key(layer),
                                                                                 ex.kv_cache.value(layer)))
                    ops.paged_append(None, key, value, None, position, sequence, cache.table, None,
                                     *cache.layer(layer))
            except BaseException:
                cache.free([slot])
                raise
            finally:
                ex.kv_cache.clear()
        return state.logits.view(-1)

    def fork(self, parents, children):
        parents, children = _slots(parents, self.device), _slots(children, self.device)
        self.cache.fork(parents, children)
        # a refused fork (cache.status, on the device) may name slots that do not exist: it indexes
        # existing ones and leaves their tokens
        source, target = (slots.clamp(0, self.sequences - 1).long() for slots in (parents, children))
        self.tokens[target] = torch.where(self.cache.status == 0, self.tokens[source], self.tokens[target])

    def free(self, slots):
        self.cache.free(slots)

    # ------------------------------------------------------------------ steps
    def _layers(self):
        ex, cache, rows = self.executor, self.cache, self.sequences
        res, eps, scale = ex.resident, ex.eps, 128 ** -0.5
        split = 1 < rows <= _SPLIT_K_MAX_TOKENS
        for index, unit in enumerate(self.runtime.plan.units):
            views = self.runtime.unit_views(index)
            layer = unit.layer_index
            w = lambda name: views[_matrix_key(layer, name)]  # noqa: B023,E731
            for operation in _UNIT_OPS.get(unit.operation, (unit.operation,)):
                if operation == "qkv":
                    ops.rmsnorm(self._x, res["model.layers.{}.input_layernorm.weight".format(layer)], eps, self._xn)
                    for name, out in (("q_proj", self._q), ("k_proj", self._k), ("v_proj", self._v)):
                        ops.gemm_bf16(self._xn, w(name), out)
                    q = self._q.view(rows, 32, 128)
                    ops.paged_append(q, self._k.view(rows, 8, 128), self._v.view(rows, 8, 128), ex.inv_freq,
                                     self._position, None, cache.table, q, *cache.layer(layer))
                elif operation == "o_proj":
                    ops.paged_attention(self._q.view(rows, 32, 128), *cache.layer(layer), cache.table, cache.lengths,
                                        scale, self._attn.view(rows, 32, 128), None, self._attention_ws)
                    ops.gemm_residual(self._attn, w("o_proj"), self._x, self._x)
                elif operation == "gate_up":
                    ops.rmsnorm(self._x, res["model.layers.{}.post_attention_layernorm.weight".format(layer)], eps,
                                self._xn)
                    ops.gemm_swiglu(self._xn, w("gate_proj"), w("up_proj"), self._mlp)
                elif operation == "down_proj":
                    if split:  # the registration lives for this launch only: it is process-wide
                        ex._register_split_k()
                    try:
                        ops.gemm_residual(self._mlp, w("down_proj"), self._x, self._x)
                    finally:
                        if split:
                            _native.lib().cb_set_gemm_workspace(None, 0, None, 0)
                else:
                    raise ValueError("the paged decoder needs the matrix_group or layer granularity (got {})".format(
                        operation))

    def _step(self):
        ex, cache = self.executor, self.cache
        full = cache.lengths >= cache.max_length  # stops alone: a reserve is all or nothing
        self._full.logical_or_(full)
        self._extra.copy_((cache.lengths > 0) & ~full)
        cache.reserve(self._extra)
        # a refused reserve leaves the lengths as they were: nothing may be written then
        went = (cache.status == 0) & (self._extra > 0)
        self._position.copy_(torch.where(went, cache.lengths - 1, -1))
        ops.embedding(self.tokens, ex.resident["model.embed_tokens.weight"], self._x)
        self._layers()
        ops.rmsnorm(self._x, ex.resident["model.norm.weight"], ex.eps, self._xn)
        ops.gemm_bf16(self._xn, ex.resident["lm_head.weight"], self.logits)
        self.logits.masked_fill_(~went.unsqueeze(1), float("nan"))

    def step(self):
        """Append every slot's token (``tokens``) to its sequence; the logits
        behind them, bf16 [sequences, vocab] (the next step's go to the same
        memory).

        Slots that took no step have NaN logits, from which :meth:`sample`
        leaves their tokens as they are: empty ones, those at ``max_length``,
        and all of them where pages ran out. Such a step can be taken again
        once pages are free; :meth:`check_errors` tells of it."""

        with torch.cuda.device(self.device), torch.inference_mode():
            if not self.use_graphs:
                self._step()
            else:
                if self._graph is None:
                    # (capture only records: the state is as before it)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        self._step()
                    self._graph = graph
                self._graph.replay()
        return self.logits

    def sample(self, logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
        """The next token of every slot into ``tokens`` (and its log probability
        into ``logprobs``) from uniform numbers in [0, 1); parameters: one value
        for all slots, or one per slot. A slot whose logits leave no choice
        (all NaN or -inf) keeps its token, at a log probability of -inf;
        :meth:`check_errors` raises if it holds a sequence."""

        def per_slot(value, dtype):
            if value is None:
                return None
            value = torch.as_tensor(value, dtype=dtype, device=self.device)
            return value.expand(self.sequences).contiguous() if value.dim() == 0 else value

        with torch.cuda.device(self.device), torch.inference_mode():
            ops.sample(logits, per_slot(temperature, torch.float32), per_slot(top_k, torch.int32),
                       per_slot(top_p, torch.float32), per_slot(min_p, torch.float32), uniform, self._picked,
                       self.logprobs)
            none = self._picked < 0
            self._no_choice.logical_or_(none & (self.cache.lengths > 0))
            self.tokens.copy_(torch.where(none, self.tokens, self._picked))
        return self.tokens, self.logprobs

    def check_errors(self):
        """Raise if a step ran out of pages or found a sequence at
        ``max_length``, a sequence had no token to choose from, or a kernel
        reported a bad index."""

        full, no_choice = (flags.nonzero().flatten().tolist() for flags in (self._full, self._no_choice))
        self._full.zero_()
        self._no_choice.zero_()
        self.cache.check()
        self.executor.check_errors()
        if full:
            raise ValueError("slots {} took no step: they hold max_length={} tokens".format(
                full, self.cache.max_length))
        if no_choice:
            raise RuntimeError("slots {} had no token to choose from: all logits NaN or -inf".format(no_choice))

    def best_of(self, prompt_ids, new_tokens, generator=None, temperature=1.0, top_k=None, top_p=None, min_p=None):
        """`sequences` sampled continuations of one prompt: (tokens int64
        [sequences, new_tokens], log probabilities fp32 of the same shape: among the
        tokens kept, after temperature and filters, so 0 where one is kept). The
        prompt's full pages are shared; every slot must be empty and is empty
        again at the end, also of a call that fails."""

        if new_tokens < 1:
            raise ValueError("new_tokens must be positive")
        used = self.cache.lengths.nonzero().flatten().tolist()
        if used:
            raise ValueError("best_of needs every slot: {} are in use".format(used))
        others = list(range(1, self.sequences))
        tokens, logprobs = [], []
        filters = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        uniform = torch.empty(self.sequences, device=self.device)
        try:
            logits = self.add(prompt_ids, 0).view(1, -1).expand(self.sequences, -1)
            if others:
                self.fork([0] * len(others), others)
                self.cache.check()
            for i in range(new_tokens):
                uniform.uniform_(generator=generator)
                picked, probability = self.sample(logits, uniform, **filters)
                tokens.append(picked.clone())
                logprobs.append(probability.clone())
                if i + 1 < new_tokens:
                    logits = self.step()
            self.check_errors()
        finally:
            self.free(list(range(self.sequences)))
        return torch.stack(tokens, 1), torch.stack(logprobs, 1)
