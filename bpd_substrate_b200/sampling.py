"""The choice of a token from a row of logits that lies on the device, by temperature, top-k, top-p and min-p (``bpd_sample_cuda``)."""
import ctypes as C
from dataclasses import dataclass
from numbers import Integral

import numpy as np

from . import capi


@dataclass(frozen=True)
class Sampling:
    """How a request's tokens are chosen.  The random numbers come from ``seed`` alone: one per token, whatever else is generated beside it."""
    temperature: float = 1.0     # 0: the largest logit
    top_k: int = 0               # 0: all
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not 0 <= self.temperature < float("inf"):
            raise ValueError(f"a temperature of {self.temperature}")
        if not 0 <= self.top_k < 2 ** 31:
            raise ValueError(f"top_k of {self.top_k}: a number of tokens, or 0 for all")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p of {self.top_p}: a share of (0, 1]")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p of {self.min_p}: a share of [0, 1]")
        if not isinstance(self.seed, Integral) or self.seed < 0:
            raise ValueError(f"a seed of {self.seed}: a whole number from 0 on")

    def numbers(self):
        """A generator of the request's random numbers, `random(dtype=np.float32)` for each token."""
        return np.random.Generator(np.random.PCG64(self.seed))


class _Row(C.Structure):
    """What goes to the device for a row, and what comes back."""
    _fields_ = [("temperature", C.c_float), ("top_k", C.c_int32), ("top_p", C.c_float), ("min_p", C.c_float), ("u", C.c_float), ("logprob", C.c_float),
                ("token", C.c_longlong)]


class TokenSampler:
    """One row at a time, on a stream of the caller's."""

    def __init__(self, lib, stream):
        self.lib, self.stream = lib, stream
        self.device, self.host = lib.bpdq_alloc(C.sizeof(_Row)), lib.bpdq_host_alloc(C.sizeof(_Row))
        if not self.device or not self.host:
            self.close()
            raise MemoryError("no room for a sampled row")
        self.row = _Row.from_address(self.host)

    def pick(self, logits, vocab, rule, u):
        """The token of fp32 logits[vocab] (a device address) for the random number u; waits for it.  -1: no logit is above -inf."""
        r, d = self.row, self.device
        r.temperature, r.top_k, r.top_p, r.min_p, r.u = rule.temperature, rule.top_k, rule.top_p, rule.min_p, u
        capi.check(self.lib.bpdq_h2d_async(d, self.host, _Row.logprob.offset, self.stream))
        at = lambda name: d + getattr(_Row, name).offset
        capi.check(self.lib.bpd_sample_cuda(logits, capi.TYPE_F32, vocab, 1, vocab, at("temperature"), at("top_k"), at("top_p"), at("min_p"), at("u"), at("token"),
                                            at("logprob"), self.stream), "bpd_sample_cuda")
        capi.check(self.lib.bpdq_d2h_async(self.host, d, C.sizeof(_Row), self.stream))
        capi.check(self.lib.bpdq_stream_sync(self.stream))
        return int(r.token)

    def close(self):
        if self.device:
            self.lib.bpdq_free(self.device)
        if self.host:
            self.lib.bpdq_host_free(self.host)
        self.device = self.host = None
