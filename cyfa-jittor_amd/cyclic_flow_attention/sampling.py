"""The choice of the next tokens of a batch of sequences, on the model's GPU:
penalties, biases and masks on the logits, then temperature, top-k, top-p and
min-p (ops.adjust_logits, ops.sample_tokens), with the sequences' tokens kept on
the device. (generation.py:23-62 of Chyxx/CyFA-Jittor v0.1.2 chooses on the
host, by temperature and top-p alone.)"""

import copy
from dataclasses import dataclass

import torch

from .ops.sampling import adjust_logits, sample_tokens


@dataclass(frozen=True)
class Sampling:
    """How tokens are chosen. Numbers are for every sequence, tensors [B] for
    each; their meaning is that of ops.adjust_logits and ops.sample_tokens.
    ``bias``: a float tensor [V] or [B, V]; ``token_bias``: a dict {token: value};
    ``allowed``: a mask (bool [V] or [B, V], or int32 words of bits), or in
    generate and generate_batch a function of the sequences' new tokens so far
    (a list of lists) that returns one, or None. ``seed``: of the batch's random
    numbers."""

    temperature: float | torch.Tensor = 1.0
    top_k: int | torch.Tensor = 0
    top_p: float | torch.Tensor = 1.0
    min_p: float | torch.Tensor = 0.0
    repetition: float | torch.Tensor = 1.0
    presence: float | torch.Tensor = 0.0
    frequency: float | torch.Tensor = 0.0
    bias: torch.Tensor | None = None
    token_bias: dict | None = None
    allowed: object = None
    seed: int = 42


class Sampler:
    """Chooses the next tokens of B sequences under a ``Sampling`` and keeps their
    tokens: ``prompts`` [B, T], of which the first ``lengths`` [B] (all without)
    count, and up to ``room`` tokens more. Its calls can be captured into a HIP
    graph (GraphedDecodeStep does), where ``generator`` has to be registered and
    the caller counts the replays with ``take``. A sequence that had no next token
    at a choice, because the mask left none or the logits held a NaN, is ``stuck``
    from then on: the token answered there is none that could follow."""

    def __init__(self, sampling, prompts, room, lengths=None):
        if prompts.dim() != 2 or prompts.dtype not in (torch.int64, torch.int32) or room < 0:
            raise ValueError("a Sampler needs prompts [B, T] of int64 or int32 tokens and room for no fewer than 0 more")
        dev, (B, T) = prompts.device, prompts.shape
        if not (sampling.allowed is None or callable(sampling.allowed) or isinstance(sampling.allowed, torch.Tensor)):
            raise ValueError(f"a Sampling's mask (allowed) must be a tensor or a function that returns one, got {type(sampling.allowed).__name__}")
        self.sampling, self.room = sampling, room
        self._follows = sampling.allowed is not None and not isinstance(sampling.allowed, torch.Tensor)  # the tokens
        self.history = torch.full((B, T + room), -1, dtype=torch.int64, device=dev)
        self.history[:, :T] = prompts
        if lengths is None:
            lengths = torch.full((B,), T, dtype=torch.int64, device=dev)
        elif lengths.shape != (B,) or lengths.dtype not in (torch.int64, torch.int32) or bool(((lengths < 0) | (lengths > T)).any()):
            raise ValueError(f"a Sampler's lengths must be {B} integers from 0 to {T}")
        self.prompt_lengths = lengths.to(device=dev, dtype=torch.int64).clone()
        self.lengths = self.prompt_lengths.clone()
        self._least = torch.full((B, 1), float("inf"), device=dev)  # of the chosen tokens' logits: -inf or NaN where none could follow
        self.generator = torch.Generator(device=dev).manual_seed(sampling.seed)

        def here(v):
            return v.to(dev) if isinstance(v, torch.Tensor) else v

        s = sampling
        self._choice = dict(temperature=here(s.temperature), top_k=here(s.top_k), top_p=here(s.top_p), min_p=here(s.min_p))
        self._penalties = dict(repetition=here(s.repetition), presence=here(s.presence), frequency=here(s.frequency))
        self._bias = here(s.bias)
        self._allowed = here(s.allowed)
        self._token_bias = None
        if s.token_bias:
            self._token_bias = (torch.tensor(list(s.token_bias), dtype=torch.int64, device=dev),
                                torch.tensor([float(v) for v in s.token_bias.values()], device=dev))
        self._penalised = any(isinstance(v, torch.Tensor) or v != none for v, none in
                              zip((s.repetition, s.presence, s.frequency), (1.0, 0.0, 0.0)))

    def __deepcopy__(self, memo):
        """A Sampler of its own state (the random numbers' among it), for a trial run."""
        other = copy.copy(self)
        other.history, other.lengths, other._least = self.history.clone(), self.lengths.clone(), self._least.clone()
        other.generator = torch.Generator(device=self.generator.device)
        other.generator.set_state(self.generator.get_state())
        return other

    def take(self):
        """Counts one token of every sequence; ValueError where there is no room for it."""
        if self.room <= 0:
            raise ValueError("the Sampler has no room for more tokens")
        self.room -= 1

    def choose(self, logits, allowed=None):
        """The next tokens [B] for logits [B, V], kept as the sequences' last; the
        caller has counted them (``take``). ``allowed`` in place of the Sampling's."""
        if allowed is None:
            if self._follows:
                raise ValueError("the Sampling's mask follows the tokens: next takes them, or choose the mask")
            allowed = self._allowed
        return self._choose(logits, allowed)

    @torch.no_grad()
    def _choose(self, logits, allowed):
        if logits.dim() != 2 or logits.shape[0] != self.history.shape[0]:
            raise ValueError(f"a Sampler of {self.history.shape[0]} sequences needs their logits [B, V], got {tuple(logits.shape)}")
        if allowed is not None:
            allowed = allowed.to(logits.device)
        if self._penalised or self._bias is not None or self._token_bias is not None or allowed is not None:
            given = (self.history, self.lengths, self.prompt_lengths) if self._penalised else (None, None, None)
            logits = adjust_logits(logits, *given, **self._penalties, bias=self._bias, token_bias=self._token_bias, allowed=allowed)
        # A number in [0, 1) and one of 2^-24 of that beside it: the first alone is 0, which takes the first kept token
        # however unlikely that is, once in 2^24 or 2^25 draws, and near 1 passes over shares below 2^-24.
        high, low = torch.rand(2, logits.shape[0], device=logits.device, generator=self.generator)
        uniform = high.double().add_(low, alpha=2.0**-24)
        ids = sample_tokens(logits, uniform, **self._choice).ids
        chosen = ids[:, None]
        torch.minimum(self._least, logits.gather(1, chosen).float(), out=self._least)  # (a NaN stays)
        at = self.lengths.clamp(max=self.history.shape[1] - 1)[:, None]
        self.history.scatter_(1, at, chosen)
        self.lengths.add_(1)
        return ids

    def next(self, logits, generated=None):
        """take and choose, with a mask from the Sampling's function of ``generated``."""
        if self._follows and generated is None:
            raise ValueError("the Sampling's mask follows the tokens: next needs the sequences' new ones")
        self.take()
        try:
            return self._choose(logits, self.sampling.allowed(generated)) if self._follows else self.choose(logits)
        except Exception:  # (a choice that is refused has taken no room)
            self.room += 1
            raise

    @property
    def stuck(self):
        """bool [B]: the sequences that had no next token at a choice so far."""
        return ~(self._least[:, 0] > float("-inf"))  # (a logit of +inf, as of a bias that forces a token, is taken)

    def to_list(self, tokens, ended=None):
        """Tokens [B] that choose or next gave, on the host; ValueError where a
        sequence is stuck that has not ``ended`` (a truth value each), -1 where it has."""
        tokens = torch.where(self.stuck, -1, tokens).tolist()
        self.check([t < 0 and (ended is None or not ended[n]) for n, t in enumerate(tokens)])
        return tokens

    @staticmethod
    def check(stuck):
        """ValueError with the first of the sequences that are ``stuck`` (truth values)."""
        for n, s in enumerate(stuck):
            if s:
                raise ValueError(f"sequence {n} has no next token: its mask leaves none, or its logits hold a NaN or nothing but -inf")
