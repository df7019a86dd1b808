"""Operators behind the vocabulary head: log probabilities of given tokens, with entropy and top alternatives."""

from .logprobs import TokenLogprobs, rl_infctx_head_token_logprobs

__all__ = ["TokenLogprobs", "rl_infctx_head_token_logprobs"]
