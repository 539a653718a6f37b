"""Refusals of the scoring calls and options that need no GPU."""
import asyncio

import pytest


class _NoModel:
    """A model that must not be touched."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} of the model was used")


def test_loops_without_log_probabilities_refuse_the_option():
    """Only generate_tokens_device returns them; the others say so instead of leaving them out."""
    from minisample import generation as G

    for n in (0, 5):
        opts = {"maxNewTokens": 2, "logprobs": n}
        for call in (lambda: G.generate_tokens(_NoModel(), [1], opts),
                     lambda: G.generate_tokens_batch(_NoModel(), [[1], [2]], opts),
                     lambda: asyncio.run(G.generate_async(_NoModel(), [1], opts))):
            with pytest.raises(ValueError, match="generate_tokens_device"):
                call()
    with pytest.raises(AssertionError):  # None is no such request
        G.generate_tokens(_NoModel(), [1], {"maxNewTokens": 2, "logprobs": None})
