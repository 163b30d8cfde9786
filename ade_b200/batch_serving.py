"""Serving many requests at once, each with its own length and its own fine-tuned model of one base.

``MultiDeltaLinear`` keeps one base weight and the deltas of several fine-tuned models (``kernels.bank_deltas``);
``attach_multi_deltas`` gives a model such modules; ``BatchDecoder`` decodes greedily for up to `max_requests` requests on a paged
key-value cache, a step of all of them replayed from one CUDA graph: page allocation (``paged_extend``), the layers with the cache write and
the attention over pages (``paged_write``, ``paged_attn_decode``), and the next tokens with their log probabilities
(``token_logprobs``).  Requests enter (``add``), leave (``finish``) and differ in length and model without a new capture.

The reference serves one delta per process and one batch of equal lengths at a time (src/serving.py:133-194, src/evaluate.py:241).
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .decode_ops import SILU_TYPES, add_rmsnorm, rmsnorm, silu_mul, token_logprobs
from .kernels import BANK_KEYS, bank_deltas, multi_delta_forward, pack_int4
from .paged import MAX_REQUESTS, paged_attn_decode, paged_extend, paged_write
from .serving import LINEAR_MODULE_NAMES, _decoder_layers

MAX_TOKENS = 128               # rows of one launch of multi_delta_forward


class DeltaRoute:
    """The fine-tuned model of every token row of the current forward, shared by the modules of a model: `ids` (rows,) int32 on the
    device, -1 for the base model, or None: the base model for every row; `models`: how many fine-tuned models there are."""

    def __init__(self, models: int):
        self.models = models
        self.ids: torch.Tensor | None = None


class MultiDeltaLinear(nn.Module):
    """W_b x + b + U_d^ (V_d^^T x) with the delta d of each row's own fine-tuned model (bfloat16, inference): the library GEMM for the
    shared term, as the reference's module has it above its own launch (src/serving.py:106-111), and one
    ``multi_delta_forward`` for every 128 rows."""

    def __init__(self, W_b: torch.Tensor, stored_forms, route: DeltaRoute, bias: torch.Tensor | None = None):
        """
        Parameters:
            W_b: base weight (d_o, d_i).
            stored_forms: for each fine-tuned model its ``pack_int4`` result for this module on the CUDA device, or None where the
                model has no delta here.
            route: the rows' models.
            bias: the base's bias (d_o,), which all of the models share, or None.
        """
        super().__init__()
        self.out_features, self.in_features = W_b.shape
        bank = bank_deltas(stored_forms)
        if (bank["M"], bank["N"]) != tuple(W_b.shape):
            raise ValueError(f"deltas are {bank['M']} x {bank['N']}, base weight {tuple(W_b.shape)}")
        self.register_buffer("weight", W_b.detach().to(device=bank["start"].device, dtype=torch.bfloat16).contiguous())
        if bias is not None and bias.shape != W_b.shape[:1]:
            raise ValueError(f"base weight is {tuple(W_b.shape)}, bias {tuple(bias.shape)}")
        self.register_buffer("bias", None if bias is None else bias.detach().to(device=self.weight.device, dtype=torch.bfloat16).contiguous())
        for k in BANK_KEYS:
            self.register_buffer(f"bank_{k}", bank[k])
        self.route = route

    def bank(self) -> dict:
        return {**{k: getattr(self, f"bank_{k}") for k in BANK_KEYS}, "M": self.out_features, "N": self.in_features}

    def forward(self, x):
        """x (..., d_i) -> (..., d_o) in bfloat16; the route names as many rows as x has."""
        x2 = x.reshape(-1, x.shape[-1]).to(torch.bfloat16).contiguous()
        y = F.linear(x2, self.weight, self.bias)
        ids = self.route.ids
        if ids is not None and x2.shape[0]:
            if ids.shape[0] != x2.shape[0]:
                raise ValueError(f"the route names {ids.shape[0]} rows, the input has {x2.shape[0]}")
            bank = self.bank()
            parts = [multi_delta_forward(a, b, bank, i) for a, b, i in zip(x2.split(MAX_TOKENS), y.split(MAX_TOKENS), ids.split(MAX_TOKENS))]
            y = parts[0] if len(parts) == 1 else torch.cat(parts)
        return y.reshape(*x.shape[:-1], self.out_features)


def attach_multi_deltas(model, base_state_dict: dict, per_model, device="cuda") -> int:
    """Give every linear module for which one of the fine-tuned models has a packed delta a MultiDeltaLinear in its place.

    `per_model` is a sequence with one mapping per fine-tuned model from ``model.layers.<i>.<name>`` to the packed fields
    (what ``attach_kernel_linears`` takes for one); `base_state_dict` maps ``model.layers.<i>.<name>.weight`` to the base weight.
    A module with a bias keeps it: ``model.layers.<i>.<name>.bias`` of `base_state_dict`, or where that has none the module's own.
    The model's route (``model._ade_route``) says which row uses which; it starts at the base model.  Returns the number of
    modules replaced.
    """
    per_model = list(per_model)
    route = model._ade_route = DeltaRoute(len(per_model))
    swapped = 0
    for li, layer in enumerate(_decoder_layers(model)):
        for sub in LINEAR_MODULE_NAMES:
            prefix = f"model.layers.{li}.{sub}"
            fetch = [d.module if hasattr(d, "module") else d.__getitem__ for d in per_model]
            forms = [pack_int4(f(prefix), device=device) if prefix in d else None for f, d in zip(fetch, per_model)]
            if all(f is None for f in forms):
                continue
            owner_path, _, leaf = sub.rpartition(".")
            owner = layer.get_submodule(owner_path)
            bias = getattr(getattr(owner, leaf), "bias", None)
            if bias is not None and prefix + ".bias" in base_state_dict:
                bias = base_state_dict[prefix + ".bias"]
            setattr(owner, leaf, MultiDeltaLinear(base_state_dict[prefix + ".weight"], forms, route, bias))
            swapped += 1
    return swapped


def _unheard(mod) -> bool:
    """Nobody would notice that `mod` is not called for a step: no forward hooks of its own or for all modules, and the forward it came with or
    ``enable_fused_decode_ops`` gave it.  The hooks with which transformers collects hidden states, once it was asked for them, stay on the
    modules and do nothing in other calls."""
    m = torch.nn.modules.module
    hooks = [h for d in (mod._forward_hooks, mod._forward_pre_hooks, m._global_forward_hooks, m._global_forward_pre_hooks) for h in d.values()]
    own = mod.__dict__
    stock = lambda f: f is None or (getattr(f, "__func__", None) is type(mod).forward and f.__self__ is mod)
    forward = own.get("forward")
    return (all(getattr(h, "__module__", None) == "transformers.utils.output_capturing" for h in hooks)
            and (stock(own.get("_ade_orig_forward")) if forward is own.get("_ade_forward") else stock(forward)))


class BatchDecoder:
    """Greedy decoding of many requests of a transformers LLaMA causal LM in bfloat16 on a CUDA device.

    Linear modules may be MultiDeltaLinear (each request then has a model of its own), ADEKernelLinear or plain.  Device state of a
    request: its length, its row of the block table, its last token, and its history: `tokens` (max_requests, max_len) and `logprobs`, the
    log probability each generated token had.  Keys of a prompt are rotated by the model's forward (bfloat16, three roundings), those of
    generated tokens by ``paged_write`` (float32, one rounding).  The step is captured at the first call of ``step``: the model's modules and weights stay as they are
    from then on.  A step calls the embedding, the rotary embedding, the linear modules and the head, whose hooks run when it is captured and
    not when it is replayed; it does the work of the other modules itself, so those have to be transformers' own and without hooks.
    """

    def __init__(self, model, max_requests: int, max_len: int, pages: int | None = None, page_size: int = 64):
        """
        Parameters:
            max_requests: requests at a time, up to 4096.
            max_len: tokens of a request, prompt and answer; rounded up to whole pages for requests that are stepped one by one.
            pages: pages of the cache; default: enough for every request at its full length.
            page_size: tokens per page.
        """
        from transformers.models.llama import modeling_llama as ml

        if not isinstance(model, ml.LlamaForCausalLM):
            raise ValueError("BatchDecoder: a LLaMA causal LM is expected")
        self.model = model
        self._check_modules()
        if model.model.rotary_emb.rope_type in ("dynamic", "longrope"):
            raise ValueError("BatchDecoder: rotary angles that change with the length would need the keys of a request anew")
        if not 1 <= max_requests <= MAX_REQUESTS or max_len < 1 or page_size < 1:
            raise ValueError(f"BatchDecoder: 1 to {MAX_REQUESTS} requests, max_len and page_size of at least 1")
        cfg = model.config
        head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        if head_dim % 32 or not 32 <= head_dim <= 256:
            raise ValueError(f"BatchDecoder: head dimensions that are a multiple of 32 up to 256 are expected; the model has {head_dim}")
        w = model.model.embed_tokens.weight
        if w.dtype != torch.bfloat16 or not w.is_cuda:
            raise ValueError("BatchDecoder: the model must be in bfloat16 on a CUDA device")
        dev, R = w.device, max_requests
        self.max_requests, self.max_len, self.page_size, self.device = R, max_len, page_size, dev
        self.heads, self.kv_heads, self.head_dim = cfg.num_attention_heads, cfg.num_key_value_heads, head_dim
        width = -(-max_len // page_size)
        pages = R * width if pages is None else int(pages)
        shape = (pages, self.kv_heads, page_size, self.head_dim)
        layers = min(cfg.num_hidden_layers, len(model.model.layers))            # the model runs the first num_hidden_layers of its layers
        self.k_pages = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(layers)]
        self.v_pages = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(layers)]
        i32 = lambda n, v=0: torch.full((n,), v, dtype=torch.int32, device=dev)
        self.block_table = torch.full((R, width), -1, dtype=torch.int32, device=dev)
        self.free_pages, self.free_count = torch.arange(pages, dtype=torch.int32, device=dev), i32(1, pages)
        self.lengths, self.new_tokens, self.status = i32(R), i32(R), i32(R)
        # one row more than there are requests takes what rows without a request produce; a history has room for what the table has room for
        self._tok = torch.zeros(R + 1, dtype=torch.long, device=dev)
        self._model_of = i32(R + 1, -1)
        self._tokens = torch.zeros(R + 1, width * page_size + 1, dtype=torch.long, device=dev)
        self._logprobs = torch.zeros(R + 1, width * page_size + 1, dtype=torch.float32, device=dev)
        self._eos = torch.full((R + 1,), -1, dtype=torch.long, device=dev)       # each request's own end token, -1: none
        self._route = getattr(model, "_ade_route", None)
        self._rows = i32(R, -1)                     # the route of a step's rows
        self._free_slots = list(range(R - 1, -1, -1))
        self._graph = None

    def _check_modules(self) -> None:
        """Refuse a model whose modules do something that a step, which does not call them, would not do."""
        from transformers.models.llama import modeling_llama as ml

        passed_by = [("the model", self.model, ml.LlamaForCausalLM), ("model", self.model.model, ml.LlamaModel), ("model.norm", self.model.model.norm, ml.LlamaRMSNorm)]
        for i, layer in enumerate(self.model.model.layers):
            passed_by.append((f"model.layers.{i}", layer, ml.LlamaDecoderLayer))
            passed_by += [(f"model.layers.{i}.{n}", getattr(layer, n, None), cls) for n, cls in
                          (("self_attn", ml.LlamaAttention), ("mlp", ml.LlamaMLP), ("input_layernorm", ml.LlamaRMSNorm), ("post_attention_layernorm", ml.LlamaRMSNorm))]
        dev = self.model.model.embed_tokens.weight.device
        for name, mod, cls in passed_by:
            if not isinstance(mod, cls) or type(mod).forward is not cls.forward or not _unheard(mod):
                raise ValueError(f"BatchDecoder: {name} has hooks or a forward of its own, which a step would not call")
            if cls is ml.LlamaRMSNorm and (mod.weight.dtype != torch.bfloat16 or mod.weight.device != dev or not mod.weight.is_contiguous()):
                raise ValueError(f"BatchDecoder: {name} must be in bfloat16 on {dev}, not {mod.weight.dtype} on {mod.weight.device}")
            if cls is ml.LlamaMLP and not (type(mod.act_fn).__name__ in SILU_TYPES and _unheard(mod.act_fn)):
                raise ValueError(f"BatchDecoder: MLPs with SiLU are expected, without hooks; {name} has {type(mod.act_fn).__name__}")

    @property
    def tokens(self) -> torch.Tensor:
        """(max_requests, max_len) token ids of every request, meaningful up to its length and the token behind it."""
        return self._tokens[:-1, :self.max_len]

    @property
    def logprobs(self) -> torch.Tensor:
        """(max_requests, max_len) log probabilities of the generated tokens, 0 for prompts."""
        return self._logprobs[:-1, :self.max_len]

    def _record(self, row, at, logits):
        """The likeliest next token of each row of logits, as the last token of request `row` and at `at` of its history."""
        _, _, logp, best = token_logprobs(logits, None, 1)
        nxt, logp = best[:, 0], logp[:, 0]
        self._tok[row] = nxt
        self._tokens[row, at] = nxt
        self._logprobs[row, at] = logp
        return nxt

    def _plain(self, *tensors):
        """What a module returned, if the launches, which take it by its address, can read it."""
        for t in tensors:
            if t.dtype != torch.bfloat16 or t.device != self.device or t.stride(-1) != 1:
                raise ValueError(f"BatchDecoder: modules that return bfloat16 on {self.device} are expected; one returned {t.dtype} on {t.device}")
        return tensors if len(tensors) > 1 else tensors[0]

    def _forward_step(self):
        R, m, lm = self.max_requests, self.model, self.model.model
        slots, positions, requests, _, _, status = paged_extend(self.lengths, self.new_tokens, self.block_table, self.free_pages, self.free_count, R,
                                                                self.page_size, in_place=True)
        self.status.copy_(torch.where(self.new_tokens > 0, status, self.status))      # a request that found its page is well again
        row = torch.where(requests < 0, R, requests).long()
        self._rows.copy_(self._model_of[row])
        x = self._plain(lm.embed_tokens(self._tok[row]))
        cos, sin = (t[0].contiguous() for t in lm.rotary_emb(x[None], positions[None]))
        layers = lm.layers[:len(self.k_pages)]
        norms = [layer.input_layernorm for layer in layers[1:]] + [lm.norm]
        h = rmsnorm(x, layers[0].input_layernorm.weight, layers[0].input_layernorm.variance_epsilon)
        for layer, nxt, kp, vp in zip(layers, norms, self.k_pages, self.v_pages):
            a, post = layer.self_attn, layer.post_attention_layernorm
            q, k, v = (p(h).view(R, -1, self.head_dim) for p in (a.q_proj, a.k_proj, a.v_proj))
            paged_write(k, v, slots, kp, vp, cos, sin)
            ctx = paged_attn_decode(q, self.block_table, requests, positions, kp, vp, a.scaling, cos, sin)
            x, h = add_rmsnorm(self._plain(a.o_proj(ctx)), x, post.weight, post.variance_epsilon)
            act = silu_mul(*self._plain(layer.mlp.gate_proj(h), layer.mlp.up_proj(h)))
            x, h = add_rmsnorm(self._plain(layer.mlp.down_proj(act)), x, nxt.weight, nxt.variance_epsilon)
        nxt = self._record(row, positions + 1, m.lm_head(h))
        # a request that has produced the end token rests
        stop = torch.cat((self.new_tokens, self.new_tokens[:1]))
        stop[row] = (nxt != self._eos[row]).int()
        self.new_tokens.copy_(torch.minimum(self.new_tokens, stop[:R]))

    @torch.no_grad()
    def step(self) -> None:
        """One token for every request whose `new_tokens` is 1; no host synchronisation once the first call has captured the step."""
        self._check_route()
        with torch.cuda.device(self.device):
            if self._graph is None:
                self._graph = self._capture()
            self._graph.replay()

    def _check_route(self) -> None:
        if getattr(self.model, "_ade_route", None) is not self._route:
            raise ValueError("BatchDecoder: the model was given other deltas since; it needs a decoder of its own for them")

    def _capture(self):
        self._check_modules()
        keep = self.new_tokens.clone()
        self.new_tokens.zero_()                     # warm-up and capture run without requests
        ids, route = None, self._route
        if route is not None:
            ids, route.ids = route.ids, self._rows
        try:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self._forward_step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._forward_step()
        finally:
            if route is not None:
                route.ids = ids
            self.new_tokens.copy_(keep)
        return graph

    def _extend(self, request: int, new: int, rows: int):
        """paged_extend for one request alone."""
        grow = torch.zeros_like(self.lengths)
        grow[request] = new
        return paged_extend(self.lengths, grow, self.block_table, self.free_pages, self.free_count, rows, self.page_size, in_place=True)

    @torch.no_grad()
    def add(self, prompt: torch.Tensor, model_id: int = -1, eos_token_id: int | None = None) -> int:
        """Enter a request: run its prompt (token ids, at least one) through fine-tuned model `model_id` (-1: the base model), keep its keys
        and values, and choose its first token.  With `eos_token_id` the request rests once it has produced that token.  Returns the
        request's number; raises when no request or page is free.  Synchronises."""
        T = int(prompt.numel())
        if not 1 <= T < self.max_len:
            raise ValueError(f"a prompt has 1 to {self.max_len - 1} tokens")
        if not -1 <= model_id < (self._route.models if self._route is not None else 0):
            raise ValueError(f"there is no fine-tuned model {model_id}")
        if not self._free_slots:
            raise ValueError(f"all {self.max_requests} requests are taken")
        self._check_route()
        words = self.model.model.embed_tokens.weight.shape[0]
        if int(prompt.min()) < 0 or int(prompt.max()) >= words:
            raise ValueError(f"a prompt's token ids are 0 to {words - 1}")
        dev, route = self.device, self._route
        with torch.cuda.device(dev):
            ids = prompt.reshape(1, T).to(device=dev, dtype=torch.long)
            b = self._free_slots[-1]
            slots, _, _, _, _, status = self._extend(b, T, T)
            state = int(status[b])
            if state:
                raise _lib.AdeKernelError(f"request {b}: {_lib.PAGED_STATUS[state]}")
            try:
                if route is not None:
                    before, route.ids = route.ids, None if model_id < 0 else torch.full((T,), model_id, dtype=torch.int32, device=dev)
                try:
                    out = self.model(input_ids=ids, use_cache=True, logits_to_keep=1)
                finally:
                    if route is not None:
                        route.ids = before
                for layer, kp, vp in zip(out.past_key_values.layers, self.k_pages, self.v_pages):
                    paged_write(layer.keys[0].transpose(0, 1), layer.values[0].transpose(0, 1), slots, kp, vp)
                self._model_of[b] = model_id
                self._eos[b] = -1 if eos_token_id is None else eos_token_id
                self._tokens[b, :T], self._logprobs[b] = ids[0], 0.0
                self._record(torch.tensor([b], device=dev), T, out.logits[:, -1])
                self.new_tokens[b] = (self._tok[b] != self._eos[b]).int()
            except BaseException:
                self._release(b)
                raise
        self._free_slots.pop()
        return b

    def _release(self, request: int) -> None:
        """Hand a request's pages back and leave nothing of it behind."""
        self._extend(request, -1, 0)
        self.new_tokens[request] = self.status[request] = 0
        self._model_of[request] = -1

    @torch.no_grad()
    def finish(self, request: int) -> None:
        """Give a request's pages and number back."""
        if request in self._free_slots or not 0 <= request < self.max_requests:
            raise ValueError(f"request {request} is not running")
        with torch.cuda.device(self.device):
            self._release(request)
        self._free_slots.append(request)

    def check_status(self) -> None:
        """Raise if a request could not grow when it last was to: no page was left, or it reached max_len.  Synchronises."""
        self._report(range(self.max_requests))

    def _report(self, requests) -> None:
        state = self.status.tolist()
        bad = [(b, state[b]) for b in requests if state[b]]
        if bad:
            raise _lib.AdeKernelError("; ".join(f"request {b}: {_lib.PAGED_STATUS[s]}" for b, s in bad))

    def generate(self, prompts, max_new_tokens: int, models=None, eos_token_id: int | None = None):
        """Answers of `max_new_tokens` tokens to a list of prompts, each by its own fine-tuned model (default: the base model), all at once.

        Returns a list of (token ids of prompt and answer, log probabilities of the answer's tokens).  With `eos_token_id` an answer ends
        with that token.  Requests that are running already rest meanwhile and go on with the next ``step``; whether they could grow
        plays no part here.
        """
        models = [-1] * len(prompts) if models is None else list(models)
        if len(models) != len(prompts) or max_new_tokens < 1:
            raise ValueError("one model for each prompt, and at least one new token")
        if any(int(p.numel()) + max_new_tokens > self.max_len for p in prompts):
            raise ValueError(f"prompt and answer have at most {self.max_len} tokens")
        if len(prompts) > len(self._free_slots):
            raise ValueError(f"{len(prompts)} prompts for {len(self._free_slots)} free requests")
        running, others = [], self.new_tokens.clone()
        try:
            self.new_tokens.zero_()
            for p, d in zip(prompts, models):
                running.append(self.add(p, d, eos_token_id))
            for _ in range(max_new_tokens - 1):
                self.step()
            self._report(running)
            out = []
            for b, p in zip(running, prompts):
                T = int(p.numel())
                n = int(self.lengths[b]) + 1          # the last token is not in the cache yet
                out.append((self._tokens[b, :n].clone(), self._logprobs[b, T:n].clone()))
            return out
        finally:
            for b in running:
                self.finish(b)
            self.new_tokens.copy_(others)
