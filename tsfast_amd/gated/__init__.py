"""Operators of a gated recurrent block: the recurrence with a matrix state per head, in training and
token by token, the norms with its gate and residual scale, and the feed-forward block behind it."""

from .core import gated_feed_forward, gated_norm, gated_recurrence, gated_recurrence_step, residual_norm  # noqa: F401
