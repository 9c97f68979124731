"""Token sampling over last-token logits (the reference leaves this to HF ``generate`` / DeepSpeed-MII)."""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Union

import torch


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool ``[n, vocab]`` -> int32 ``[n, words]``: bit v % 32 of word v // 32 is token v's."""
    n, V = allowed.shape
    bits = torch.zeros(n, -(-V // 32) * 32, dtype=torch.int64, device=allowed.device)
    bits[:, :V] = allowed
    words = (bits.view(n, -1, 32) << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


class LogitControls:
    """What the requests of a batch lay on their logits from step to step: penalties for repeated tokens, a bias per token, a mask of the
    tokens that a grammar allows next. ``prompts[i]``: the tokens of request i so far (of a session, its earlier turns' too); numbers and dicts are for all requests, lists of them for
    each. ``ops.kernels.logit_controls`` has the formulas."""

    def __init__(self, prompts: Sequence, vocab: int, max_new_tokens: int, device, repetition_penalty: Union[float, Sequence[float]] = 1.0,
                 presence_penalty: Union[float, Sequence[float]] = 0.0, frequency_penalty: Union[float, Sequence[float]] = 0.0,
                 logit_bias: Union[None, Dict[int, float], Sequence[Optional[Dict[int, float]]]] = None, allowed: Optional[torch.Tensor] = None) -> None:
        n, self.vocab, self.device = len(prompts), vocab, torch.device(device)
        told = [torch.as_tensor(p).reshape(-1).to(torch.int32).cpu() for p in prompts]
        each = lambda v, name: self._each(v, n, name)  # noqa: E731
        rep, pres, freq = each(repetition_penalty, "repetition_penalty"), each(presence_penalty, "presence_penalty"), each(frequency_penalty, "frequency_penalty")
        if any(not 0 < r < math.inf for r in rep):
            raise ValueError("repetition_penalty must be positive and finite in 32 bits")
        if not all(map(math.isfinite, pres + freq)):
            raise ValueError("presence_penalty and frequency_penalty must be finite in 32 bits")
        self._c = {}
        self._room = 0
        if any(r != 1 for r in rep) or any(pres) or any(freq):
            history = torch.full((n, max((t.numel() for t in told), default=0) + max_new_tokens), -1, dtype=torch.int32)
            for i, t in enumerate(told):
                history[i, :t.numel()] = t
            lengths = torch.tensor([t.numel() for t in told], dtype=torch.int32)
            f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
            self._c = {"history": history, "history_len": lengths, "prompt_len": lengths.clone(), "repetition": f(rep), "presence": f(pres),
                       "frequency": f(freq)}
            self._room = max_new_tokens
        if logit_bias:
            lists = [logit_bias] * n if isinstance(logit_bias, dict) else [b or {} for b in logit_bias]
            if len(lists) != n:
                raise ValueError(f"logit_bias is for {len(lists)} requests, there are {n}")
            k = max(map(len, lists), default=0)
            if any(not 0 <= t < vocab for b in lists for t in b):
                raise ValueError("logit_bias names a token outside the vocabulary")
            bias = torch.tensor([list(b.values()) + [0.0] * (k - len(b)) for b in lists], dtype=torch.float32).reshape(n, k)
            if not (bias < math.inf).all():
                raise ValueError("logit_bias must be finite in 32 bits, or -inf")
            self._c["bias_ids"], self._c["bias"] = torch.tensor([list(b) + [-1] * (k - len(b)) for b in lists], dtype=torch.int32).reshape(n, k), bias
        self._c = {name: t.to(self.device) for name, t in self._c.items()}
        self.n = n
        self.set_allowed(allowed)

    @staticmethod
    def _each(value, n: int, name: str) -> List[float]:
        values = [float(v) for v in value] if isinstance(value, (list, tuple)) else [float(value)] * n
        if len(values) != n:
            raise ValueError(f"{name} is for {len(values)} requests, there are {n}")
        return torch.tensor(values, dtype=torch.float32).tolist()       # as the kernel has them: 1e39 is infinite, 1e-46 nothing

    def set_allowed(self, allowed: Optional[torch.Tensor]) -> None:
        """The tokens that may come next: bool ``[n, vocab]``, or None for all. Stays until the next call."""
        if allowed is None:
            self._c.pop("mask", None)
            return
        if allowed.dtype != torch.bool or tuple(allowed.shape) != (self.n, self.vocab):
            raise ValueError(f"allowed must be bool {(self.n, self.vocab)}, got {allowed.dtype} {tuple(allowed.shape)}")
        self._c["mask"] = pack_mask(allowed.to(self.device))

    def apply(self, logits: torch.Tensor) -> torch.Tensor:
        """New logits; the given ones are left as they are."""
        if tuple(logits.shape) != (self.n, self.vocab):
            raise ValueError(f"logits must be {(self.n, self.vocab)}, got {tuple(logits.shape)}")
        if not self._c or not self.n:
            return logits
        from ..ops.backend import get_ops
        return get_ops(logits.device).logit_controls(logits, torch.empty_like(logits, memory_format=torch.contiguous_format), **self._c)

    def append(self, tokens: torch.Tensor) -> None:
        """The tokens that the requests have been given, ``[n]``."""
        if tokens.numel() != self.n:
            raise ValueError(f"{tokens.numel()} tokens for {self.n} requests")
        if "history" not in self._c or not self.n:
            return
        if self._room < 1:
            raise RuntimeError("more tokens than max_new_tokens")
        self._room -= 1
        at = self._c["history_len"]
        self._c["history"].scatter_(1, at[:, None].long(), tokens.reshape(-1, 1).to(self.device, torch.int32))
        at += 1

    def keep(self, places: Sequence[int]) -> None:
        """The requests that go on, by their places among the present ones."""
        places = list(places)
        if places == list(range(self.n)):
            return
        if any(not 0 <= p < self.n for p in places):       # (on a GPU the index itself would end the context)
            raise ValueError(f"places {places} of {self.n} requests")
        at = torch.tensor(places, dtype=torch.int64, device=self.device)
        self._c = {name: t[at] for name, t in self._c.items()}
        self.n = len(places)


def _drawable(logits: torch.Tensor) -> torch.Tensor:
    """Logits whose softmax is a distribution whatever the controls left of them (drawing from anything else ends a GPU's context): an infinite one
    is the largest there is, and a row without any token has token 0, as the arg-max has it. Rows whose largest logit may leave 32 bits when it is divided by
    a temperature have it taken off."""
    x = torch.nan_to_num(logits.float(), nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    x[:, 0] = torch.where(x.amax(-1) == -math.inf, 0.0, x[:, 0])
    top = x.amax(-1, keepdim=True)
    return x - torch.where(top.abs() > 1e30, top, 0.0)


def sample_next(logits: torch.Tensor, do_sample: bool = False, temperature: float = 1.0, top_k: int = 0,
                top_p: float = 1.0, controls: Optional[LogitControls] = None) -> torch.Tensor:
    """``logits [n, vocab]`` -> int32 ``[n]``. Greedy decoding runs the library's arg-max kernel on a GPU. ``controls`` are laid on the logits first,
    and told the tokens."""
    if controls is not None:
        left = controls.apply(logits)
        tokens = sample_next(_drawable(left) if do_sample and temperature != 0.0 else left, do_sample, temperature, top_k, top_p)
        controls.append(tokens)
        return tokens
    if not do_sample or temperature == 0.0:
        if logits.device.type == "cuda" and logits.dtype in (torch.bfloat16, torch.float16, torch.float32):
            from ..ops import kernels
            return kernels.argmax(logits.contiguous())
        return logits.float().argmax(-1).to(torch.int32)
    if math.isnan(temperature) or top_p < 0.0:       # (they would leave no distribution, and drawing from none ends a GPU's context)
        raise ValueError(f"temperature is {temperature} and top_p {top_p}")
    x = logits.float() / min(max(temperature, 1e-6), 1e30)       # (-inf stays that)
    if top_k and top_k > 0:
        kth = torch.topk(x, min(top_k, x.shape[-1]), dim=-1).values[..., -1:]
        x = x.masked_fill(x < kth, float("-inf"))
    if top_p < 1.0:
        sorted_x, idx = torch.sort(x, descending=True, dim=-1)
        probs = torch.softmax(sorted_x, dim=-1)
        cum = probs.cumsum(-1)
        drop = cum - probs > top_p
        sorted_x = sorted_x.masked_fill(drop, float("-inf"))
        x = torch.full_like(x, float("-inf")).scatter(-1, idx, sorted_x)
    return torch.multinomial(torch.softmax(x, dim=-1), 1).squeeze(-1).to(torch.int32)
