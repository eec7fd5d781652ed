"""One step of a beam search on the MI355X: selection over beams x vocabulary, and the states in their new order.

``KerasRNNTDecoder.beam_search`` (reference rnnt/rnnt_decoder.py:95-233) adds a hypothesis's score to the log-probabilities
of its inner step and keeps the best candidates, one hypothesis at a time on the host.  ``beam_select`` does a whole batch
of beams in one or two launches straight from the joint's logits (log-softmax included, see also ``joint_log_softmax``);
``beam_reorder`` gathers every state tensor of the hypotheses in one more.
"""
from __future__ import annotations

from . import _lib


def beam_select(logits, scores, width, enc=None, allowed=None, finished=None, end=0):
    """The `width` best continuations of every utterance's beams.

    logits [B, K, V] (float32, bfloat16 or float16): the joint's output for K hypotheses, or, with enc [B, V] of the same
    type, the prediction network's part of an additive joint (logits + enc, rounded to float32, as joint_log_softmax does).
    scores [B, K] float32: log-probabilities so far; -inf, NaN or anything beyond +-2^30 marks an empty beam.
    allowed: bool [V] or [B, V]; a forbidden symbol is no candidate and has no part in the softmax, whatever its logit.
    finished: bool [B, K]; such a beam is carried along, as one candidate with its own score at symbol `end`, allowed or not (in
    a transducer: a hypothesis that has emitted blank and waits for the next frame).  Nothing is differentiable here.

    Returns scores [B, width] float32, parent [B, width] int32 (beam) and token [B, width] int32, in descending order of
    scores + log_softmax (compared in float64, where a row's log sum exp is good to 2^-21.6: its terms are float32), ties to the lowest
    beam, then the lowest symbol.  Where there are fewer
    candidates than `width`: -inf, -1, -1.  A beam whose allowed logits hold NaN or +inf, or nothing above -inf, has none."""
    return _lib.native().beam_select(logits, scores, width, enc, allowed, finished, end)


def beam_reorder(parent, states, batch_dim=0, out=None):
    """Network states, token histories, lengths ... of the hypotheses beam_select kept.

    parent: int32 [B, W] as beam_select returns it.  states: a list of tensors of any type whose dimensions batch_dim and
    batch_dim + 1 are (B, K) -- [layers, B, K, hidden] has batch_dim 1.  Returns a list with W in the place of K and row
    parent[b, w] of utterance b at [b, w]; zeros where parent is -1 (any value outside [0, K)).  out: tensors to write to
    instead of new ones, dense, of the results' shapes and types, sharing no memory with states or one another, and
    requiring no gradients.  Nothing is differentiable here."""
    return _lib.native().beam_reorder(parent, states, batch_dim, out)
