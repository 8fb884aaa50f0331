"""Helpers shared by evaluation and sampling: rebuild a model from a checkpoint, score a split, generate text.

Evaluation and probes load only the consolidated ``model.pt`` export into a plain (unwrapped) model, whatever
strategy trained it (the reference's experiment layer does the same: scripts/synbios_moe.py:141-168).
"""

from __future__ import annotations

import math
from pathlib import Path
from typing import Any

import torch

from mini_train_sys_b200.models import MiniTransformer, ModelConfig, get_ops_backend
from mini_train_sys_b200.train.checkpoint import load_model_state_dict_from_checkpoint


def model_config_from_checkpoint(path: str | Path) -> dict[str, Any] | None:
    runtime = Path(path) / "runtime.pt"
    if not runtime.is_file():
        return None
    blob = torch.load(runtime, map_location="cpu", weights_only=False)
    cfg = (blob.get("config") or {}).get("model")
    return dict(cfg) if cfg else None


def load_model_for_inference(checkpoint: str | Path, *, model_payload: dict[str, Any] | None = None, ops: str = "torch",
                             device: torch.device | str = "cpu", dtype: torch.dtype = torch.float32) -> MiniTransformer:
    payload = model_payload or model_config_from_checkpoint(checkpoint)
    if not payload:
        raise ValueError("no model config given and none recorded in the checkpoint")
    model = MiniTransformer(ModelConfig(**payload), get_ops_backend(ops), activation_dtype=dtype)
    state = load_model_state_dict_from_checkpoint(checkpoint)
    missing, unexpected = model.load_state_dict(state, strict=False)
    missing = [k for k in missing if not (k == "lm_head.weight" and model.cfg.tie_word_embeddings)]
    if missing or unexpected:
        raise ValueError(f"checkpoint does not match the model: missing={missing[:4]} unexpected={unexpected[:4]}")
    return model.to(device).eval()


@torch.no_grad()
def evaluate_loss(model: MiniTransformer, loader, device: torch.device, *, max_batches: int | None = None,
                  autocast_dtype: torch.dtype | None = None) -> dict[str, float]:
    """Token-weighted mean cross entropy and perplexity over ``loader``."""

    total, tokens, batches = 0.0, 0, 0
    for batch in loader:
        ids, tgt = batch["input_ids"].to(device), batch["targets"].to(device)
        with torch.autocast(device.type, dtype=autocast_dtype, enabled=autocast_dtype is not None):
            hidden = model.hidden_states(ids)
            loss = model.ops.fused_linear_cross_entropy(hidden.reshape(-1, hidden.shape[-1]), model.lm_head.weight, tgt.reshape(-1))
        n = int((tgt != -100).sum())
        total += float(loss) * n
        tokens += n
        batches += 1
        if max_batches is not None and batches >= max_batches:
            break
    mean = total / max(tokens, 1)
    return {"loss": mean, "perplexity": math.exp(min(mean, 50.0)), "tokens": tokens, "batches": batches}


KV_CACHES = ("none", "int8")


# operators whose plain forms ask the device for numbers, which a captured step cannot
_CAPTURED_OPS = ("kv_append", "cached_attention", "moe_tokens", "fused_moe")


class DecodeSession:
    """Cached decoding of one batch: ``prompt`` once, then ``step`` by step.

    On a GPU with the native operators a step is captured into a CUDA graph after the first one over a filled cache and replayed: a
    step is some hundred short kernels, whose launches take longer than their work.  ``cache.reset()`` starts anew.  Where the kernels do not cover the model (a head dimension
    other than 32, 64 and 128, ...) steps stay eager, or are refused with ``graph=True``.  Weights that change in place or move are
    noticed, and the step is captured again; a model whose parameters are replaced by others needs a new session.

    A native kernel that gives up on a wait computes on without what it waited for and raises its device's status word.  The word is
    copied to the host behind every call, without waiting, and the next call raises RuntimeError if it was set; ``check()`` waits and
    looks at once (``generate`` does so at its end)."""

    def __init__(self, model: MiniTransformer, batch: int, capacity: int | None = None, *, graph: bool | None = None) -> None:
        self.model = model
        model.check_decodable()
        self.cache = model.new_cache(batch, capacity)
        on_gpu = self.cache.device.type == "cuda" and getattr(model.ops, "name", "") == "native" and model.activation_dtype == torch.bfloat16
        if graph and not on_gpu:
            raise ValueError("a captured step needs a GPU, the native operators and bf16 activations")
        self.graph_wanted = on_gpu if graph is None else bool(graph)
        self._insisted = bool(graph)
        self._graph: torch.cuda.CUDAGraph | None = None
        self._prepared = False
        self._status = self._status_word()
        self._seen = None if self._status is None else torch.zeros_like(self._status, device="cpu", pin_memory=self._status.is_cuda)

    def _status_word(self) -> torch.Tensor | None:
        """Where the kernels of this session report, None where it runs none."""

        if self.cache.device.type != "cuda" or getattr(self.model.ops, "name", "") != "native":
            return None
        from mini_train_sys_b200.ops.native_backend import ext

        return ext().status_tensor(self.cache.device.index)

    def _note_status(self) -> None:
        if self._status is None or (self._status.is_cuda and torch.cuda.is_current_stream_capturing()):
            return
        if self._status.is_cuda:
            with torch.cuda.device(self._status.device):
                self._seen.copy_(self._status, non_blocking=True)
        else:
            self._seen.copy_(self._status)

    def _raise_noted(self) -> None:
        if self._seen is not None and int(self._seen[0]) != 0:
            self.check()

    def check(self) -> None:
        """Raise if a kernel of this session gave up on a wait (synchronises)."""

        if self._status is not None:
            from mini_train_sys_b200.ops.native_backend import raise_status

            raise_status(int(self._status[0].item()))

    def prompt(self, input_ids: torch.Tensor, counts: torch.Tensor | None = None) -> torch.Tensor:
        """Logits [B, V] behind the prompts [B, T]; ``counts`` [B] are their lengths where they are padded on the right."""

        self._raise_noted()
        logits = self.model.decode(input_ids, self.cache, counts)
        self._note_status()
        return logits

    def step(self, token_ids: torch.Tensor) -> torch.Tensor:
        """Logits [B, V] behind one more token [B, 1] of every sequence.  They are overwritten by the next step."""

        self._raise_noted()
        logits = self._step(token_ids)
        self._note_status()
        return logits

    def _step(self, token_ids: torch.Tensor) -> torch.Tensor:
        if token_ids.shape != (self.cache.batch, 1):
            raise ValueError(f"a step takes one token per sequence, got {tuple(token_ids.shape)}")
        if not self.graph_wanted or self.cache.held == 0:          # nothing is cached: the form of a prompt, which no later step takes
            return self.model.decode(token_ids, self.cache)
        if self._graph is not None and self._weights() != self._captured:
            self._graph, self._prepared = None, False
        if not self._prepared:
            return self._eager_step(token_ids)
        if self.cache.held + 1 > self.model.rotary.max_seq_len:
            raise ValueError(f"{self.cache.held} cached + 1 new tokens exceed the model's seq_len of {self.model.rotary.max_seq_len}")
        if self._graph is None:
            self._capture(token_ids)
        if self.model.training:
            raise RuntimeError("decode() needs eval mode")
        if any(m._forward_hooks or m._forward_pre_hooks for m in self._modules):
            self.model.check_decodable()
        self.cache.replayed(1)
        with torch.cuda.device(self.cache.device):             # on that device's current stream, behind the copy
            self._ids.copy_(token_ids)
            self._graph.replay()
        return self._logits

    def _eager_step(self, token_ids: torch.Tensor) -> torch.Tensor:
        """The step before a capture: it lays out what the kernels keep, and shows whether they cover the model."""

        def plain_calls() -> int:
            return sum(self.model.ops.dispatch[f"{op}:fallback"] for op in _CAPTURED_OPS)

        before = plain_calls()
        logits = self.model.decode(token_ids, self.cache)
        if plain_calls() != before:
            if self._insisted:
                raise ValueError("the native kernels do not cover this model: its steps cannot be captured")
            self.graph_wanted = False
        self._prepared = True
        return logits

    def _capture(self, token_ids: torch.Tensor) -> None:
        from mini_train_sys_b200.ops.native_backend import kept_bf16

        self._ids = token_ids.clone()
        self._modules = list(self.model.blocks.modules())
        self._tensors = [*self.model.parameters(), *self.model.buffers()]
        held = self.cache.held
        torch.cuda.synchronize(self.cache.device)
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.device(self.cache.device), torch.cuda.graph(graph):
                self._logits = self.model.decode(self._ids, self.cache)
        finally:
            self.cache.held, self.cache.padded = held, None        # capturing has run nothing
        self._copies = [kept_bf16(t) for t in self._tensors]           # the graph reads them: not to be freed while it lives
        self._captured = self._weights()
        self._graph = graph

    def _weights(self) -> list[tuple[int, int]]:
        """Addresses and versions of the weights: a graph reads them where they were, and bf16 copies of fp32 ones as they were."""

        return [(t.data_ptr(), 0 if t.is_inference() else t._version) for t in self._tensors]


def _next_token(logits: torch.Tensor, temperature: float, top_k: int | None, greedy: bool, generator) -> torch.Tensor:
    step = logits.float()
    if greedy or temperature <= 0:
        return step.argmax(-1, keepdim=True)
    step = step / temperature
    if top_k is not None and top_k > 0:
        kth = step.topk(min(top_k, step.shape[-1]), -1).values[:, -1:]
        step = step.masked_fill(step < kth, float("-inf"))
    return torch.multinomial(torch.softmax(step, -1), 1, generator=generator)


@torch.no_grad()
def generate(model: MiniTransformer, prompt_ids: torch.Tensor, *, max_new_tokens: int, temperature: float = 1.0,
             top_k: int | None = None, greedy: bool = False, generator: torch.Generator | None = None, kv_cache: str = "none") -> torch.Tensor:
    """Autoregressive decoding.  Without a cache the prefix (cropped to ``seq_len``) is re-encoded every step; with
    ``kv_cache="int8"`` every token is encoded once and finished blocks of 64 keys and values are held in 8 bits, and prompt and
    new tokens together must fit in ``seq_len``."""

    if kv_cache not in KV_CACHES:
        raise ValueError(f"kv_cache must be one of {KV_CACHES}, got {kv_cache!r}")
    ids = prompt_ids.clone()
    limit = model.cfg.seq_len
    if kv_cache == "none":
        for _ in range(max_new_tokens):
            _, logits = model(ids[:, -limit:])
            ids = torch.cat((ids, _next_token(logits[:, -1, :], temperature, top_k, greedy, generator)), dim=1)
        return ids
    if max_new_tokens <= 0:
        return ids
    reach = ids.shape[1] + max_new_tokens - 1                  # the last token is not fed back
    if reach > limit:
        raise ValueError(f"{ids.shape[1]} prompt + {max_new_tokens} new tokens exceed the model's seq_len of {limit}; cached decoding does not crop")
    session = DecodeSession(model, ids.shape[0], reach)
    logits = session.prompt(ids)
    for i in range(max_new_tokens):
        nxt = _next_token(logits, temperature, top_k, greedy, generator)
        ids = torch.cat((ids, nxt), dim=1)
        if i + 1 < max_new_tokens:
            logits = session.step(nxt)
    session.check()
    return ids
