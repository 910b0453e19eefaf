"""Next tokens of a batch whose rows each bring their own settings (``n730_sample_rows``).

Addresses are device addresses as ints (0: none), one value a row: temperature, top_k, top_p and min_p
(0: none of that cut, temperature 1), u (numbers in [0, 1) that the caller draws), tokens out.  Raises
``N730Error`` on a negative code; ``include/n730_cuda.h`` has the rule.
"""
from __future__ import annotations

from . import _lib
from .kv8 import DTYPES


def sample_rows(logits: int, dtype: str, batch: int, vocab: int, u: int, tokens: int, *, ld: int = 0, temperature: int = 0,
                top_k: int = 0, top_p: int = 0, min_p: int = 0, prob: int = 0, kept: int = 0, stream: int = 0):
    """tokens[row] from the row's logits; prob: the token's share of the kept mass, kept: how many tokens were."""
    _lib.check(_lib.cuda().n730_sample_rows(logits, DTYPES[dtype], batch, vocab, ld or vocab, temperature, top_k, top_p, min_p, u,
                                            tokens, prob, kept, stream), "sample_rows")
